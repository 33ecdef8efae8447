"""PyTorch-facing ops: the reference's ``forward`` signature plus the BASELINE ``forward_lse``.

These call the in-tree extension ``nsa_hopper_b200._C`` (nsa_sel_torch.cpp), which calls the C
ABI of ``libnsa_sel.so``.  There is no CPU or eager fallback: if the extension or the library
is missing, or the device is not a B200, the call raises.
"""
from __future__ import annotations

import math
from fractions import Fraction
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

try:
    from . import _C  # type: ignore[attr-defined]
except ImportError as e:  # pragma: no cover - exercised only when the build is missing
    raise ImportError("nsa_hopper_b200._C is not built: run `python -m nsa_hopper_b200.build`") from e


def forward(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, sel: torch.Tensor, l_prime: int, BQ: int,
            cyc: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Drop-in for the reference op ``mod.forward(Q,K,V,sel,l_prime,BQ,cyc)`` (nsa_v2.cu:147):
    returns fp32 O [B,Hq,S,D].  ``cyc`` may be an int64 CUDA tensor of NQB*B*Hkv*2 entries
    (accumulated into) or empty/None."""
    if cyc is None:
        cyc = torch.empty(0, dtype=torch.int64, device=Q.device)
    return _C.forward(Q, K, V, sel, int(l_prime), int(BQ), cyc)


def forward_lse(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, sel: torch.Tensor, l_prime: int = 64,
                BQ: int = 1, cu_seqlens: Optional[torch.Tensor] = None, scale: float = 0.0,
                out_f32: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Selected-branch forward returning (O bf16 [B,Hq,T,d_v], LSE fp32 [B,Hq,T])."""
    o, lse = _C.forward_lse(Q, K, V, sel, int(l_prime), int(BQ), cu_seqlens, float(scale), bool(out_f32))
    return o, lse


def forward_ext(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, sel: torch.Tensor, l_prime: int = 64, BQ: int = 1,
                window: int = 0, key_map: int = 0, scale: float = 0.0, out: Optional[torch.Tensor] = None,
                weight: Optional[torch.Tensor] = None, accumulate: bool = False,
                with_lse: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """Forward with extended key visibility (fp32 O, fp32 LSE): ``window`` > 0 limits query t to
    keys p with t - p < window; ``key_map`` = 1 treats K/V as compressed keys (kv_len rows) visible
    to t iff float32 linspace(0, T-1, kv_len)[i] <= t (the compressed branch of NSA).

    Fused output combination: the result is multiplied by ``weight[0]`` (an fp32 CUDA tensor, read
    on the device) and written to ``out``, or added into it when ``accumulate`` (TMA reduce-add),
    so the NSA gate g_c*O_cmp + g_s*O_sel + g_w*O_win is three launches into one buffer.
    ``with_lse=False`` skips the LSE (an empty tensor is returned in its place)."""
    o, lse = _C.forward_ext(Q, K, V, sel, int(l_prime), int(BQ), int(window), int(key_map), float(scale), out, weight,
                            bool(accumulate), bool(with_lse))
    return o, lse


def select_blocks(Q: torch.Tensor, K: torch.Tensor, n_sel: int, l_prime: int = 64, cmp_block: int = 32,
                  cmp_stride: int = 16) -> torch.Tensor:
    """Block selection on the GPU (nsa_sel_select): int32 [B, Hkv, T, min(n_sel, ceil(T/l_prime))],
    best block first, -1 where fewer blocks are visible (reference nsa_reference.py:27-44)."""
    return _C.select_blocks(Q, K, int(n_sel), int(l_prime), int(cmp_block), int(cmp_stride))


def backward(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, sel: torch.Tensor, O: torch.Tensor,
             LSE: torch.Tensor, dO: torch.Tensor, l_prime: int = 64, scale: float = 0.0
             ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients (fp32 dQ, dK, dV) of the selected-branch forward for the upstream gradient dO,
    given that forward's O (bf16 or fp32) and LSE.  Per-token selection (sel [B,Hkv,T,KSEL]),
    d = 128, G = Hq/Hkv in {8, 16} (nsa_sel_backward; the reference has no backward pass).  The
    workspace comes from torch's caching allocator; the library allocates nothing."""
    from . import capi

    for name, t in (("Q", Q), ("K", K), ("V", V), ("dO", dO)):
        if t.dtype != torch.bfloat16 or not t.is_cuda or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous bf16 CUDA tensor")
    if O.dtype not in (torch.bfloat16, torch.float32) or not O.is_contiguous():
        raise ValueError("O must be a contiguous bf16 or fp32 tensor")
    if LSE.dtype != torch.float32 or not LSE.is_contiguous():
        raise ValueError("LSE must be a contiguous fp32 tensor")
    sel = sel.to(torch.int32).contiguous()
    B, Hq, T, d = Q.shape
    Hkv = K.shape[1]
    dq = torch.zeros(B, Hq, T, d, device=Q.device, dtype=torch.float32)
    dk = torch.zeros(B, Hkv, T, d, device=Q.device, dtype=torch.float32)
    dv = torch.zeros_like(dk)
    desc = capi.make_bwd_desc(
        q=Q.data_ptr(), k=K.data_ptr(), v=V.data_ptr(), sel=sel.data_ptr(), o=O.data_ptr(), lse=LSE.data_ptr(),
        d_o=dO.data_ptr(), dq=dq.data_ptr(), dk=dk.data_ptr(), dv=dv.data_ptr(), batch=B, heads_q=Hq,
        heads_kv=Hkv, seq_len=T, d=d, n_sel=sel.shape[-1], block_size=int(l_prime),
        o_dtype=capi.DTYPE_BF16 if O.dtype == torch.bfloat16 else capi.DTYPE_F32, scale=float(scale))
    ws = torch.empty(capi.backward_workspace_bytes(desc), device=Q.device, dtype=torch.uint8)
    desc.workspace = ws.data_ptr()
    capi.backward(desc, torch.cuda.current_stream(Q.device).cuda_stream)
    return dq, dk, dv


class SelectedAttention(torch.autograd.Function):
    """Selected-branch attention with its backward: ``O = SelectedAttention.apply(Q, K, V, sel)``
    (per-token selection, l_prime = 64) returns bf16 O and supports ``O.backward(dO)``; Q, K, V
    receive bf16 gradients computed by nsa_sel_backward."""

    @staticmethod
    def forward(ctx, Q, K, V, sel, l_prime: int = 64):
        O, LSE = forward_lse(Q, K, V, sel, l_prime, 1)
        ctx.save_for_backward(Q, K, V, sel, O, LSE)
        ctx.l_prime = l_prime
        return O

    @staticmethod
    def backward(ctx, dO):
        Q, K, V, sel, O, LSE = ctx.saved_tensors
        dq, dk, dv = backward(Q, K, V, sel, O, LSE, dO.contiguous().to(torch.bfloat16), ctx.l_prime)
        return dq.to(Q.dtype), dk.to(K.dtype), dv.to(V.dtype), None, None


PAGE = 64  # tokens of a page of the 4-bit cache


def cache_alloc(num_pages: int, heads_kv: int, d_qk: int, d_v: int, device="cuda") -> torch.Tensor:
    """A 4-bit paged KV cache of zeros: uint8 [num_pages, heads_kv, 36 * (d_qk + d_v)], a page holding
    64 tokens (4.5 bits a value; the layout of a record is described in include/nsa_sel.h)."""
    return torch.zeros(num_pages, heads_kv, _C.cache_record_bytes(int(d_qk), int(d_v)), dtype=torch.uint8, device=device)


def cache_write(cache: torch.Tensor, K: torch.Tensor, V: torch.Tensor, pages: torch.Tensor, lens: torch.Tensor,
                cu_seqlens: Optional[torch.Tensor] = None) -> None:
    """Quantises the newest tokens of a batch of sequences into the 4-bit cache (nsa_cache_write).

    ``pages`` int32 [S, W] is the page table, ``lens`` int32 [S] the sequences' tokens, the new ones
    included.  K [N, Hkv, d_qk] and V [N, Hkv, d_v] (bf16 or fp16, any row and head strides that are
    multiples of 8) hold the rows: row r of sequence s, ``cu_seqlens[s] <= r < cu_seqlens[s + 1]``, is
    its token ``lens[s] - (cu_seqlens[s + 1] - r)``; without ``cu_seqlens`` row s is the last token of
    sequence s.  A prefill of one sequence in the forward's layout [1, Hkv, T, d] is
    ``K[0].transpose(0, 1)`` with ``cu_seqlens = [0, T]``.  Tokens that the page table does not hold
    (a page < 0, a position < 0 or behind the table) are not written, rows of no sequence neither."""
    _C.cache_write(cache, K, V, pages, lens, cu_seqlens)


def cache_read(cache: torch.Tensor, d_qk: int, pages: torch.Tensor, lens: torch.Tensor,
               cu_seqlens: Optional[torch.Tensor] = None, n_tokens: Optional[int] = None,
               dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """Reads the batch's newest tokens back from the 4-bit cache (nsa_cache_read): K [1, Hkv, N, d_qk] and
    V [1, Hkv, N, d_v], packed as ``forward_lse`` takes a varlen batch with the same ``cu_seqlens``.
    ``n_tokens`` = N is needed with ``cu_seqlens`` (whose last entry the host cannot see); a whole
    sequence is read where it has ``lens[s]`` rows.  The values are exact in every dtype; tokens that
    the page table does not hold, and rows of no sequence, are zeros."""
    if n_tokens is None:
        if cu_seqlens is not None:
            raise ValueError("n_tokens (the rows that cu_seqlens packs) is needed with cu_seqlens")
        n_tokens = lens.shape[0]
    k, v = _C.cache_read(cache, int(d_qk), pages, lens, cu_seqlens, int(n_tokens), dtype)
    return k, v


def cache_attend(Q: torch.Tensor, cache: torch.Tensor, pages: torch.Tensor, lens: torch.Tensor,
                 sel: Optional[torch.Tensor] = None, l_prime: int = 64, window: int = 0,
                 cu_seqlens: Optional[torch.Tensor] = None, scale: float = 0.0, out: Optional[torch.Tensor] = None,
                 weight: Optional[torch.Tensor] = None, accumulate: bool = False, with_lse: bool = True,
                 err: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of the batch's newest tokens over the 4-bit cache (nsa_cache_attend): the decode step.

    Q [N, Hq, d_qk] (bf16 or fp16) has the rows of :func:`cache_write`; the row at position t sees
    the keys p <= t, with ``window`` > 0 those with t - p < window, and with ``sel`` int32
    [N, Hkv, KSEL] those in its selected blocks of ``l_prime`` keys (a set; entries < 0 or behind t
    select nothing; KSEL at most 1024).  Returns (O [N, Hq, d_v] of Q's dtype, LSE fp32 [N, Hq], natural log); a row that
    sees no key, or of no sequence, has O = 0 and LSE = -inf.

    ``out``, ``weight``, ``accumulate``: as in :func:`forward_ext`, the result times ``weight[0]`` is
    written to ``out`` (fp32 or Q's dtype) or added into it (fp32); rows of no sequence are then left
    as they were.  ``with_lse=False`` skips the LSE (an empty tensor is returned).  No gradients.

    ``err`` (int32 on the device, optional): 1 is ORed into its first element if a copy inside the kernel did not come within
    2 seconds, which no correct program meets; rows that it belonged to are then NaN.  Nothing is raised, as the call does not
    wait for the device."""
    o, lse = _C.cache_attend(Q, cache, pages, lens, sel, int(l_prime), int(window), cu_seqlens, float(scale), out, weight,
                             bool(accumulate), bool(with_lse), err)
    return o, lse


class CacheBatch(NamedTuple):
    """A call's batch, as :func:`cache_reserve` works it out."""
    lens: torch.Tensor                  # int32 [S] tokens of the sequences that got rows (these included), 0 for the others
    cu_seqlens: Optional[torch.Tensor]  # int32 [S + 1] where the rows are packed (n_tokens), else None
    positions: torch.Tensor             # int32 [N] a row's position in its sequence, -1 for an absent row
    slots: torch.Tensor                 # int64 [N] PAGE * page + position % PAGE, -1 for an absent row
    held: torch.Tensor                  # int32 [S] tokens of every sequence after the call
    n_free: torch.Tensor                # int32 [1] free pages after the call


def cache_reserve(pages: torch.Tensor, held: torch.Tensor, rows: torch.Tensor, pool: torch.Tensor, n_free: torch.Tensor,
                  n_tokens: Optional[int] = None, update: bool = True) -> CacheBatch:
    """Page table, lengths, packing, positions and slots of a call's batch, from the tokens that each request gets or gives
    back (nsa_cache_reserve).  Everything is on the device: a step can be captured, and replayed with other ``rows``.

    ``pages`` int32 [S, W] is the page table, ``held`` int32 [S] the tokens that the sequences hold, ``pool`` int32 [P] the
    free pages, of which the first ``n_free`` (int32 [1]) count.  ``rows`` int32 [S]: > 0, the sequence asks for that many
    more tokens; < 0, it gives its last ones back (rejected drafts, or all of a sequence that has ended: ``-held``), and the pages
    with them; 0, it has no part in the call.  Pages that are given back come first, then those that are asked for are taken
    from the end of the pool, by the sequences in their order.  A sequence that does not fit its row of the table, or for which
    (it and those before it) the pool has too few pages, stays as it was and has no rows: its ``lens`` is 0, which the cache's
    calls take as absent rows, and ``held`` tells the scheduler.

    With ``n_tokens`` = N the call's rows are packed (``rows[s]`` for each sequence that asks, those of refused ones too, N at
    least their sum); without, row s is sequence s's last token.  Tokens that a sequence gives back and tokens that it asks for
    (rejected drafts, then new ones) take two calls.  ``pages`` and ``pool`` are changed in place, ``held`` and ``n_free`` too
    unless ``update`` is False: then new tensors are returned and nothing that counts has changed, so the call can be made
    again.  A page that two sequences share must not be given back while the other uses it."""
    lens, cu, positions, slots, held, n_free = _C.cache_reserve(pages, held, rows, pool, n_free,
                                                                None if n_tokens is None else int(n_tokens), bool(update))
    return CacheBatch(lens, None if n_tokens is None else cu, positions, slots, held, n_free)


def cache_select(Q: torch.Tensor, cmp_cache: torch.Tensor, cmp_pages: torch.Tensor, lens: torch.Tensor, n_sel: int,
                 l_prime: int = 64, cmp_block: int = 32, cmp_stride: int = 16,
                 cu_seqlens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`select_blocks` for the batch's newest tokens, from the compressed keys of a 4-bit cache (nsa_cache_select;
    ``nsa.cache_compress`` keeps them): int32 [N, Hkv, n_sel], the ``sel`` of :func:`cache_attend`.

    Q [N, Hq, d_qk] (bf16 or fp16) has the rows of :func:`cache_attend`; ``lens`` int32 [S] are the tokens of the sequences (not
    their compressed keys).  The row at position t gets what the last row of ``select_blocks`` gets for t + 1 tokens: the
    blocks of ``l_prime`` tokens with the largest sums of (summed query heads) . (compressed key), the best first, -1 behind
    the last.  Scores are compared as 64-bit sums, equal ones by the lower block; scores that are not finite come last (of a
    query that is not finite all are, so that the lowest blocks are selected).
    ``n_sel`` at most 1024, Hq / Hkv at most 256, sequences of up to 2^24 tokens (longer ones, and those whose compressed keys
    ``cmp_pages`` cannot hold, select nothing).  No gradients."""
    return _C.cache_select(Q, cmp_cache, cmp_pages, lens, int(n_sel), int(l_prime), int(cmp_block), int(cmp_stride), cu_seqlens)


class RotaryPlan(NamedTuple):
    """Which values of a head :func:`rotary` turns, and how fast (made by :func:`rotary_plan`, kept for all calls)."""
    d: int
    offset: int
    interleaved: bool
    axes: int
    turns: torch.Tensor  # int64 [pairs] on the host: inv_freq / 2 pi in units of 2^-64
    axis: torch.Tensor   # uint8 [pairs] on the host


# 2^192 / (2 pi)
_TURN = round(2**192 / (2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640629")))


def _turns(inv_freq: float) -> int:
    """inv_freq / (2 pi) in units of 2^-64, modulo a turn, as int64."""
    n, d = float(inv_freq).as_integer_ratio()
    t = (2 * n * _TURN // (d << 128) + 1) // 2 % 2**64
    return t - 2**64 if t >= 2**63 else t


def rotary_plan(d: int, *, rotary_dim: Optional[int] = None, offset: int = 0, base: float = 10000.0,
                sections: Optional[Sequence[int]] = None, interleaved: bool = False,
                inv_freq: Optional[Sequence[float]] = None, axis: Optional[Sequence[int]] = None) -> RotaryPlan:
    """How :func:`rotary` turns heads of ``d`` (at most 256) values: ``rotary_dim`` of them (all unless given) from ``offset``
    on, value i with value i + rotary_dim / 2 of that part, or neighbours (``interleaved``).

    Pair i turns by position * ``base`` ** (-2 i / rotary_dim), or position * ``inv_freq[i]`` (radians, taken in 64 bits).  With
    several axes (time, height, width) each pair follows one: ``sections`` = (16, 24, 24) gives the first 16 pairs the first
    axis and so on; ``axis`` names it pair by pair instead.  At most four axes."""
    dim = d if rotary_dim is None else rotary_dim
    if not 0 < d <= 256:
        raise ValueError("d must be from 1 to 256")
    if dim < 2 or dim % 2 or offset < 0 or offset + dim > d:
        raise ValueError("rotary_dim must be even and positive, and lie in the head with its offset")
    pairs = dim // 2
    if inv_freq is None:
        if not base > 0:
            raise ValueError("base must be positive")
        inv_freq = [float(base) ** (-i / pairs) for i in range(pairs)]
    if axis is None:
        sections = [pairs] if sections is None else list(sections)
        if any(n < 0 for n in sections) or sum(sections) != pairs:
            raise ValueError(f"sections must add up to the {pairs} pairs")
        axis, axes = [a for a, n in enumerate(sections) for _ in range(n)], len(sections)
    elif sections is not None:
        raise ValueError("sections and axis exclude each other")
    else:
        axis = [int(a) for a in axis]
        axes = max(axis, default=0) + 1
    if len(axis) != pairs or len(inv_freq) != pairs:
        raise ValueError(f"axis and inv_freq must have an entry for each of the {pairs} pairs")
    if axes > 4 or min(axis) < 0:
        raise ValueError("there are one to four axes")
    if not all(math.isfinite(f) for f in inv_freq):
        raise ValueError("inv_freq must be finite")
    return RotaryPlan(d, offset, bool(interleaved), axes,
                      torch.tensor([_turns(f) for f in inv_freq], dtype=torch.int64, device="cpu"),
                      torch.tensor(axis, dtype=torch.uint8, device="cpu"))


def rotary(Q: torch.Tensor, K: Optional[torch.Tensor], positions: torch.Tensor, plan: RotaryPlan,
           inverse: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Turns Q and K (or Q alone: ``K`` None) by their tokens' positions (nsa_rotary).

    Rows Q [N, Hq, d] and K [N, Hkv, d] as the cache's calls take them, or heads [B, Hq, T, d] and [B, Hkv, T, d] as the forward
    does; bf16, fp16 or fp32, any strides (a projection's [B, T, H, d] is given as ``x.transpose(1, 2)``).  ``positions`` int32
    [N] or [B, T] (any strides, e.g. expanded over the batch), with the axes of the plan before that if there are several.
    The results are contiguous and of the inputs' dtype.  Angles of all int32 positions are reduced to an eighth of a turn with an
    error below 2^-32 of a turn, and then rounded to fp32; sines, cosines and products are fp32.
    Differentiable in Q and K, any number of times, in reverse and in forward mode (``torch.autograd.forward_ad``; the transforms
    of ``torch.func`` are refused); ``inverse`` turns back."""
    q, k = _C.rotary(Q, K, positions, plan.turns, plan.axis, plan.axes, plan.d, plan.offset, plan.interleaved, bool(inverse))
    return q, k


def library_version() -> int:
    return int(_C.library_version())
