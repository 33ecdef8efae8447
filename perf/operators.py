"""The 4-bit paged KV cache's operators as cases to measure: their plain form in elementary torch
operations (``own = False``) and the framework's calls (``own = True``).

Three kinds of case, all on one batch description: ``pages`` int32 [S, W] (page table; a page holds 64
tokens), ``lens`` int32 [S] (tokens of each sequence, the call's rows included) and optionally ``cu``
int32 [S + 1] (packed rows; without it every sequence has one row).  Row r of sequence s is the token at
position ``lens[s] - (cu[s+1] - r)``.

* ``write``: K and V of the rows are quantised into the cache and read back (what a prefill does that goes
  on with the values that the later decode sees);
* ``read``: rows of the cache are read back, packed;
* ``attend``: every row's query attends to its sequence's cache: all keys, a window, or selected blocks.

A cache is uint8 [pages, Hkv, 36 * (d_qk + d_v)].  A record holds K codes [64][d_qk / 2], K scales
[64][d_qk / 16], V codes [64][d_v / 2] and V scales [64][d_v / 16].  Codes are E2M1 (0, 0.5, 1, 1.5, 2, 3,
4, 6 and a sign; the low nibble is the even index); a scale, one for 16 neighbouring values, has 5 exponent
bits (bias 15) and 3 mantissa bits.
"""
import math

import torch

own = False

PAGE = 64
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MAX_SCALE = 10240.0  # the largest scale whose sixfold still is a finite half-precision number
DIMS = ((64, 64), (128, 128), (192, 128), (128, 64))
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ the cases
def _case(name, kind, seqs, lo, hi, rows, hq, hkv, dims, dtype="bf16", mode="all", n_sel=0, l_prime=64, window=0, empty=0):
    """`seqs` sequences of `lo` to `hi` tokens, each with `rows` rows in the call (0: as many as it has tokens; one row
    each goes without cu_seqlens, n > 1 stands for 1 to n in turn); the first `empty` sequences have no tokens at all."""
    return {"name": name, "kind": kind, "seqs": seqs, "lo": lo, "hi": hi, "rows": rows, "hq": hq, "hkv": hkv, "d_qk": dims[0],
            "d_v": dims[1], "dtype": dtype, "mode": mode, "n_sel": n_sel, "l_prime": l_prime, "window": window, "empty": empty}


def listed():
    return [
        # one decode step's new tokens: few rows, latency
        _case("write_step_8", "write", 8, 1, 9000, 1, 64, 4, (128, 128)),
        # a large decode batch's new tokens, keys wider than values
        _case("write_step_512", "write", 512, 1, 4000, 1, 64, 4, (192, 128)),
        # a prefill of a few prompts of odd lengths into a small model's cache
        _case("write_prompts_odd", "write", 7, 129, 6001, 0, 16, 1, (64, 64), "fp16"),
        # one long prefill
        _case("write_prefill_64k", "write", 1, 65536, 65536, 0, 64, 4, (128, 128)),
        # the last 32 tokens of every sequence, for the next compressed key
        _case("read_tail_32", "read", 64, 40, 5000, 32, 64, 4, (128, 128)),
        # whole contexts of a ragged batch, to go on prefilling
        _case("read_contexts", "read", 16, 1, 12289, 0, 64, 4, (192, 128)),
        # one sequence's decode step at the framework's headline shape: latency
        _case("attend_selected_1", "attend", 1, 65536, 65536, 1, 64, 4, (128, 128), mode="selected", n_sel=16),
        # a decode batch of the same model
        _case("attend_selected_256", "attend", 256, 1, 16384, 1, 64, 4, (128, 128), mode="selected", n_sel=16),
        # a few drafted tokens a sequence, wide blocks, sequences that have ended
        _case("attend_selected_drafts", "attend", 48, 1, 20001, 4, 32, 4, (128, 64), "fp16", "selected", 8, 128, empty=3),
        # the sliding-window branch
        _case("attend_window_128", "attend", 128, 1, 8000, 1, 64, 4, (192, 128), mode="window", window=512),
        # every key: one long context
        _case("attend_all_1", "attend", 1, 131072, 131072, 1, 64, 4, (128, 128)),
        # every key: a ragged batch (also the compressed branch, whose keys are all visible)
        _case("attend_all_64", "attend", 64, 1, 32768, 1, 64, 4, (128, 128)),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("write", "read", "attend", "attend", "attend"))
    dims, dtype = rng.choice(DIMS), rng.choice(("bf16", "fp16"))
    hq, hkv = rng.choice(((64, 4), (32, 4), (16, 1), (16, 2), (8, 8), (48, 4), (28, 4), (32, 1), (5, 5)))
    if kind != "attend":
        rows = rng.choice((0, 0, 1, 5, 32))
        most = 65536 * 4 * 256 // (hkv * sum(dims))  # tokens that cost what the largest listed prefill does
        seqs = _log_int(rng, 1, 512)
        hi = _log_int(rng, 1, 65536 if rows else max(1, min(65536, most // seqs)))
        hi = max(1, min(hi, 8 * most // seqs))
        return _case("", kind, seqs, 1, hi, rows, hq, hkv, dims, dtype, empty=rng.choice((0, 0, 1)) if seqs > 1 else 0)
    mode = rng.choice(("all", "selected", "window"))
    rows = rng.choice((1, 1, 2, 4))
    most = 64 * 32768 * 4 * 256 // (hkv * sum(dims))  # tokens that cost what the largest listed case does
    seqs = _log_int(rng, 1, 256)
    hi = _log_int(rng, 1, max(1, min(131072, most // (seqs * (rows if mode == "all" else 1)))))
    n_sel = rng.choice((1, 4, 8, 16, 16, 24)) if mode == "selected" else 0
    l_prime, window = rng.choice((64, 64, 128, 256)), _log_int(rng, 1, 2048) if mode == "window" else 0
    if mode != "all":
        seqs = min(seqs, max(1, most // (2 * rows * (n_sel * l_prime + window))))
    return _case("", "attend", seqs, 1, hi, rows, hq, hkv, dims, dtype, mode, n_sel, l_prime, window,
                 rng.choice((0, 0, 1)) if seqs > 1 else 0)


def _lengths(case):
    """Tokens of each sequence, and the rows that each has in the call."""
    n, empty = case["seqs"], case["empty"]
    live = max(1, n - empty)
    lens = [0] * (n - live) + [case["lo"] + (case["hi"] - case["lo"]) * (i + 1) // live for i in range(live)]
    if case["rows"] == 0:
        return lens, list(lens)
    if case["rows"] == 1:
        return lens, [1] * n
    if case["kind"] != "attend":
        return lens, [min(case["rows"], x) for x in lens]
    return lens, [1 + i % case["rows"] for i in range(n)]


def _visible(case, pos):
    """Keys that the row at `pos` sees."""
    if pos < 0:
        return 0
    if case["mode"] == "window":
        return min(pos + 1, case["window"])
    if case["mode"] == "selected":
        lp = case["l_prime"]
        return (min(case["n_sel"], pos // lp + 1) - 1) * lp + pos % lp + 1
    return pos + 1


def work(case):
    lens, rows = _lengths(case)
    d, hq, hkv = case["d_qk"] + case["d_v"], case["hq"], case["hkv"]
    wide, held = 2 * hkv * d, 9 * hkv * d // 16  # bytes of a token outside and inside the cache
    if case["kind"] != "attend":
        n = sum(rows)
        return {"bytes": n * (wide + held + (wide if case["kind"] == "write" else 0)), "flops": n * hkv * d}
    n, keys, once = sum(rows), 0, 0
    for length, r in zip(lens, rows):
        seen = [_visible(case, length - r + i) for i in range(r)]
        keys += sum(seen)
        if case["mode"] == "selected":  # the first and the newest block are the same for a sequence's rows
            once += max(seen) + sum(max(0, x - 2 * case["l_prime"]) for x in seen[:-1])
        else:
            once += min(max(length, 0), max(seen) + (r - 1 if case["mode"] == "window" else 0))
    outside = n * hq * (2 * d + 4) + 4 * n * hkv * case["n_sel"] + 4 * once // PAGE
    return {"bytes": once * held + outside, "flops": 2 * keys * hq * d}


# ------------------------------------------------------------------ inputs
def _two_to(e):
    """fp32 2 ** e of int32 e."""
    return ((e + 127) << 23).view(torch.float32)


def _quantise(x):
    """fp32 [..., d] to codes uint8 [..., d / 2] and scales uint8 [..., d / 16]."""
    g = x.unflatten(-1, (-1, 16))
    amax = g.abs().amax(-1)
    fine = amax.isfinite()
    raw = torch.where(fine, amax, torch.zeros_like(amax)) / torch.full_like(amax, 6.0)  # (a number as divisor is multiplied by)
    step = _two_to(torch.clamp(torch.frexp(raw).exponent - 1, min=-14) - 3)
    s = torch.clamp(torch.round(raw / step) * step, max=MAX_SCALE)
    exponent = torch.clamp(torch.frexp(s).exponent - 1, min=-14)
    eighths = torch.round(s / _two_to(exponent - 3)).int()  # 8 to 15, below 8 for the smallest
    scale = torch.where(fine, (exponent + 14) * 8 + eighths, torch.full_like(eighths, 255)).to(torch.uint8)
    live = (fine & (s > 0)).unsqueeze(-1)
    y = torch.where(live, g / torch.where(s > 0, s, torch.ones_like(s)).unsqueeze(-1), torch.zeros_like(g))
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int()
            + (a > 5.0).int() + torch.signbit(y).int() * 8)
    code = code.flatten(-2)
    return (code[..., 0::2] + code[..., 1::2] * 16).to(torch.uint8), scale


def _tables(device):
    """The two values that a byte of codes stands for [256, 2], and the value of every scale byte [256], fp32."""
    value = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=device)
    byte = torch.arange(256, device=device)
    pair = torch.stack((value[byte % 16], value[byte // 16]), -1)
    scale = (byte << 7).to(torch.int16).view(torch.float16).float()
    return pair, scale


def _split(records, d_qk, d_v):
    """K codes, K scales, V codes and V scales of records uint8 [..., 36 * (d_qk + d_v)], each [..., 64, bytes]."""
    parts = torch.split(records, [PAGE * d_qk // 2, PAGE * d_qk // 16, PAGE * d_v // 2, PAGE * d_v // 16], -1)
    return [p.unflatten(-1, (PAGE, -1)) for p in parts]


def _values(codes, scales):
    """fp32 [..., d] that codes [..., d / 2] and scales [..., d / 16] stand for."""
    pair, scale = _tables(codes.device)
    v = pair.index_select(0, codes.reshape(-1).int()).view(*codes.shape[:-1], -1, 16)
    return (v * scale.index_select(0, scales.reshape(-1).int()).view(*scales.shape, 1)).flatten(-2)


def _keys_and_values(shape, d_qk, d_v, gen):
    """K with channels of unequal size, as a model's are, and V."""
    gain = torch.exp(0.5 * torch.randn(d_qk, device="cuda", generator=gen))
    k = torch.randn(*shape, d_qk, device="cuda", generator=gen) * gain
    return k, torch.randn(*shape, d_v, device="cuda", generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lens, rows = _lengths(case)
    n, hq, hkv, d_qk, d_v = sum(rows), case["hq"], case["hkv"], case["d_qk"], case["d_v"]
    dtype = DTYPES[case["dtype"]]
    order = torch.randperm(case["seqs"], device="cuda", generator=gen)
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")[order]
    rows = torch.tensor(rows, dtype=torch.int32, device="cuda")[order]
    need = (lens + PAGE - 1) // PAGE
    total, width = int(need.sum()), max(1, int(need.max()))
    # pages in an order of their own, a few of the pool in nobody's hands; -1 behind a sequence's last page
    pool = torch.randperm(total + 3, device="cuda", generator=gen)[:total].int()
    held = torch.arange(width, device="cuda") < need.unsqueeze(1)
    pages = torch.full((case["seqs"], width), -1, dtype=torch.int32, device="cuda")
    pages[held] = pool
    cache = torch.zeros(total + 3, hkv, 36 * (d_qk + d_v), dtype=torch.uint8, device="cuda")
    state = {"case": dict(case), "cache": cache, "pages": pages, "lens": lens, "n": n, "cu": None}
    if case["rows"] != 1:
        state["cu"] = torch.cat((torch.zeros(1, device="cuda"), rows.cumsum(0))).to(torch.int32)
    if case["kind"] == "write":
        k, v = _keys_and_values((n, hkv), d_qk, d_v, gen)
        return state | {"k": k.to(dtype), "v": v.to(dtype)}
    for part in cache.split(max(1, (1 << 27) // (hkv * PAGE * (d_qk + d_v)))):
        k, v = _keys_and_values((part.shape[0], hkv, PAGE), d_qk, d_v, gen)
        for x, at in ((k, 0), (v, 36 * d_qk)):
            codes, scales = _quantise(x.to(dtype).float())
            both = torch.cat((codes.flatten(-2), scales.flatten(-2)), -1)
            part[..., at:at + both.shape[-1]] = both
    if case["kind"] == "read":
        return state
    state["q"] = torch.randn(n, hq, d_qk, device="cuda", generator=gen).to(dtype)
    state["sel"] = None
    if case["mode"] == "selected":
        # the first block, the newest, and others at random, the best first; -1 where there are fewer
        _, pos, _ = _rows(state)
        k, lp = case["n_sel"], case["l_prime"]
        newest = torch.clamp(pos, min=0) // lp
        blocks = int(newest.max()) + 1
        mark = torch.rand(n, hkv, blocks, device="cuda", generator=gen)
        mark[..., 0] += 1
        mark.scatter_add_(2, newest.view(-1, 1, 1).expand(-1, hkv, 1), torch.full_like(mark[..., :1], 2.0))
        mark.masked_fill_(torch.arange(blocks, device="cuda") > newest.view(-1, 1, 1), -1.0)
        best, index = mark.topk(min(k, blocks), -1)
        sel = torch.full((n, hkv, k), -1, dtype=torch.int32, device="cuda")
        sel[..., :index.shape[-1]] = torch.where(best >= 0, index, torch.full_like(index, -1)).int()
        state["sel"] = sel
    return state


# ------------------------------------------------------------------ the plain form
def _rows(state):
    """Each row's sequence, its position, and the page and place there (page -1: no such token)."""
    row = torch.arange(state["n"], device="cuda", dtype=torch.int32)
    lens, pages, cu = state["lens"], state["pages"], state["cu"]
    if cu is None:
        seq, pos = row.long(), lens[row.long()] - 1
    else:
        seq = torch.searchsorted(cu, row, right=True) - 1
        pos = lens[seq] - (cu[seq + 1] - row)
    at = torch.clamp(pos, min=0).long()
    page = torch.where(pos >= 0, pages[seq, at // PAGE], torch.full_like(pos, -1))
    return seq, pos.long(), (page.long(), at % PAGE)


def _read(state):
    case, cache = state["case"], state["cache"]
    _, _, (page, place) = _rows(state)
    there = page >= 0
    parts = _split(cache, case["d_qk"], case["d_v"])
    kc, ks, vc, vs = (p[torch.clamp(page, min=0), :, place].transpose(0, 1) for p in parts)
    dtype = DTYPES[case["dtype"]]
    return [torch.where(there.view(-1, 1), _values(c, s), 0.0).to(dtype).unsqueeze(0) for c, s in ((kc, ks), (vc, vs))]


def _write(state):
    case = state["case"]
    _, _, (page, place) = _rows(state)
    there = page >= 0
    page, place = page[there], place[there]
    kc, ks = _quantise(state["k"][there].float())
    vc, vs = _quantise(state["v"][there].float())
    for part, x in zip(_split(state["cache"], case["d_qk"], case["d_v"]), (kc, ks, vc, vs)):
        part[page, :, place] = x


def _attend(state):
    case, q, cache, pages = state["case"], state["q"], state["cache"], state["pages"]
    n, hq, hkv, d_qk, d_v = state["n"], case["hq"], case["hkv"], case["d_qk"], case["d_v"]
    seq, pos, _ = _rows(state)
    width = pages.shape[1]
    # the 64-key sub-blocks of every row and KV head, and whether they count
    if case["mode"] == "selected":
        sel, per = state["sel"].long(), case["l_prime"] // PAGE
        twice = ((sel.unsqueeze(-1) == sel.unsqueeze(-2)).tril(-1)).any(-1)
        sub = (sel.unsqueeze(-1) * per + torch.arange(per, device="cuda")).flatten(-2)
        counts = ((sel >= 0) & ~twice).repeat_interleave(per, -1)
    elif case["mode"] == "window":
        first = torch.clamp(pos - case["window"] + 1, min=0) // PAGE
        sub = first.unsqueeze(-1) + torch.arange((case["window"] + PAGE - 2) // PAGE + 1, device="cuda")
        sub = sub.unsqueeze(1).expand(n, hkv, -1)
        counts = torch.ones_like(sub, dtype=torch.bool)
    else:
        sub = torch.arange(width, device="cuda").expand(n, hkv, width)
        counts = torch.ones_like(sub, dtype=torch.bool)
    counts = counts & (sub < width) & (sub * PAGE <= pos.view(-1, 1, 1))
    page = pages[seq.view(-1, 1, 1), torch.clamp(sub, 0, width - 1)].long()
    counts = counts & (page >= 0)
    records = cache[torch.clamp(page, min=0), torch.arange(hkv, device="cuda").view(1, -1, 1)]
    kc, ks, vc, vs = _split(records, d_qk, d_v)
    key = sub.unsqueeze(-1) * PAGE + torch.arange(PAGE, device="cuda")
    seen = counts.unsqueeze(-1) & (key <= pos.view(-1, 1, 1, 1))
    if case["mode"] == "window":
        seen = seen & (key > pos.view(-1, 1, 1, 1) - case["window"])
    seen = seen.flatten(-2).unsqueeze(2)
    k = _values(kc, ks).flatten(2, 3)
    score = torch.matmul(q.float().view(n, hkv, hq // hkv, d_qk), k.transpose(-1, -2)) / math.sqrt(d_qk)
    del k
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    del score
    total = p.sum(-1, keepdim=True)
    v = torch.where(seen.transpose(-1, -2).squeeze(2).view(n, hkv, -1, 1), _values(vc, vs).flatten(2, 3), 0.0)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    lse = top + torch.log(total)
    return o.view(n, hq, d_v).to(q.dtype), lse.view(n, hq)


def run(state):
    case = state["case"]
    if own:
        from nsa_hopper_b200 import ops

        batch = (state["pages"], state["lens"])
        if case["kind"] == "attend":
            return ops.cache_attend(state["q"], state["cache"], *batch, sel=state["sel"], l_prime=case["l_prime"],
                                    window=case["window"], cu_seqlens=state["cu"])
        if case["kind"] == "write":
            ops.cache_write(state["cache"], state["k"], state["v"], *batch, cu_seqlens=state["cu"])
        return ops.cache_read(state["cache"], case["d_qk"], *batch, cu_seqlens=state["cu"], n_tokens=state["n"],
                              dtype=DTYPES[case["dtype"]])
    if case["kind"] == "attend":
        return _attend(state)
    if case["kind"] == "write":
        _write(state)
    return _read(state)


# ------------------------------------------------------------------ the definition, in 64 bits
def _power(e):
    """fp64 2 ** e of whole fp64 e, to the bit (a power computed on the GPU is not)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _rounded(x):
    """Quantised fp64 [..., d], by the definition: the nearest scale, then the nearest multiple of it, ties to even."""
    g = x.double().unflatten(-1, (-1, 16))
    amax = g.abs().amax(-1, keepdim=True)
    raw = amax / torch.full_like(amax, 6.0)
    octave = torch.clamp(torch.floor(torch.log2(torch.clamp(raw, min=2.0 ** -40))), min=-14)
    s = torch.clamp(torch.round(raw * _power(3 - octave)) * _power(octave - 3), max=MAX_SCALE)
    y = g.abs() / torch.where(s > 0, s, 1.0)
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0)).double()
    y = torch.clamp(torch.round(y / step) * step, max=6.0) * s
    return torch.where(g < 0, -y, y).flatten(-2)


def _decoded(codes, scales):
    """fp64 values of codes and scales, from their fields."""
    nibble = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double()
    sign = 1 - 2 * torch.floor(nibble / 8)
    field = nibble % 8
    two = torch.floor(field / 2)
    size = torch.where(two == 0, field / 2, (1 + (field % 2) / 2) * _power(two - 1))
    s = scales.double()
    five = torch.floor(s / 8)
    s = torch.where(five == 0, (s % 8) * 2.0 ** -17, (8 + s % 8) * _power(five - 18))
    return sign * size * s.repeat_interleave(16, -1)


def exact(case, seed):
    state = prepare(case, seed)
    lens, pages, cache, n = state["lens"].tolist(), state["pages"], state["cache"], state["n"]
    cu = list(range(n + 1)) if state["cu"] is None else state["cu"].tolist()
    d_qk, d_v, hq, hkv = case["d_qk"], case["d_v"], case["hq"], case["hkv"]
    if case["kind"] == "write":
        ok = torch.cat([torch.arange(x - (b - a), x) >= 0 for x, a, b in zip(lens, cu, cu[1:])]).view(-1, 1, 1).cuda()
        return [torch.where(ok, _rounded(x), 0.0).transpose(0, 1).unsqueeze(0) for x in (state["k"], state["v"])]
    ks, vs = torch.zeros(hkv, n, d_qk, dtype=torch.float64, device="cuda"), torch.zeros(hkv, n, d_v, dtype=torch.float64, device="cuda")
    o = torch.zeros(n, hq, d_v, dtype=torch.float64, device="cuda")
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device="cuda")
    for s, length in enumerate(lens):
        if length == 0 or cu[s] == cu[s + 1]:
            continue
        first = 0
        if case["kind"] == "read" or case["mode"] == "window":
            first = max(0, length - (cu[s + 1] - cu[s]) - (case["window"] if case["kind"] == "attend" else 0)) // PAGE
        records = cache[pages[s, first:(length + PAGE - 1) // PAGE].long()].transpose(0, 1)
        kc, ksc, vc, vsc = _split(records, d_qk, d_v)
        k, v = _decoded(kc, ksc).flatten(1, 2), _decoded(vc, vsc).flatten(1, 2)
        base = first * PAGE
        for r in range(cu[s], cu[s + 1]) if case["kind"] == "attend" else ():
            pos = length - (cu[s + 1] - r)
            if pos < 0:
                continue
            at = torch.arange(base, base + k.shape[1], device="cuda")
            seen = (at <= pos).expand(hkv, -1)
            if case["mode"] == "window":
                seen = seen & (at > pos - case["window"])
            elif case["mode"] == "selected":
                seen = seen & torch.isin(at // case["l_prime"] + torch.arange(hkv, device="cuda").view(-1, 1) * (1 << 32),
                                         torch.where(state["sel"][r] >= 0, state["sel"][r].long() + torch.arange(
                                             hkv, device="cuda").view(-1, 1) * (1 << 32), -1))
            q = state["q"][r].double().view(hkv, hq // hkv, d_qk)
            score = torch.where(seen.unsqueeze(1), q @ k.transpose(1, 2) / math.sqrt(d_qk), -math.inf)
            lse[r] = torch.logsumexp(score, -1).view(hq)
            o[r] = (torch.softmax(score, -1) @ torch.where(seen.unsqueeze(-1), v, 0.0)).view(hq, d_v)
        if case["kind"] == "read":
            rows = cu[s + 1] - cu[s]
            skip = max(0, rows - length)
            lo = length - rows + skip - base
            ks[:, cu[s] + skip:cu[s + 1]] = k[:, lo:lo + rows - skip]
            vs[:, cu[s] + skip:cu[s + 1]] = v[:, lo:lo + rows - skip]
    return (o, lse) if case["kind"] == "attend" else [ks.unsqueeze(0), vs.unsqueeze(0)]
