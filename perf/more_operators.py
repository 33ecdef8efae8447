"""What a decode step needs around the 4-bit cache, and what comes before attention, as cases to measure: their plain form in
elementary torch operations (``own = False``) and the framework's calls (``own = True``).

* ``reserve``: page table, lengths, packing, positions and slots of a batch from the tokens that each request gets or gives
  back, with the pages taken from a pool of free ones;
* ``rotary``: Q and K turned by positions of one or several axes (time, height, width); for training with the gradients;
* ``select``: the best blocks of every new token by the scores of its query against the compressed keys of a 4-bit cache.

A page holds 64 tokens.  A cache is uint8 [pages, Hkv, 36 * (d_qk + d_v)]; a record starts with K codes [64][d_qk / 2] and K
scales [64][d_qk / 16].  Codes are E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign; the low nibble is the even index); a scale, one
for 16 neighbouring values, has 5 exponent bits (bias 15) and 3 mantissa bits.
"""
import math

import numpy as np
import torch

own = False

PAGE = 64
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DIMS = ((64, 64), (128, 128), (192, 128), (128, 64))
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
CMP_BLOCK, CMP_STRIDE = 32, 16


# ------------------------------------------------------------------ the cases
def _reserve_case(name, seqs, width, lo, hi, rows, packed, ended=0.0, idle=0.0, short=0.0):
    """`seqs` sequences that hold `lo` to `hi` tokens and get 1 to `rows` more; shares of them have ended (they give all back)
    or idle; the pool lacks the share `short` of the pages that are wanted.  `packed`: rows stand one after the other, else
    row s is sequence s's."""
    return {"name": name, "kind": "reserve", "seqs": seqs, "width": width, "lo": lo, "hi": hi, "rows": rows, "packed": packed,
            "ended": ended, "idle": idle, "short": short}


def _rotary_case(name, batch, tokens, hq, hkv, d, rotary_dim, offset, sections, interleaved, dtype="bf16", train=False,
                 base=1e6):
    """`batch` 0: rows [tokens, H, d]; else heads of [batch, tokens, H, d].  `sections`: pairs of each axis, as a text."""
    return {"name": name, "kind": "rotary", "batch": batch, "tokens": tokens, "hq": hq, "hkv": hkv, "d": d,
            "rotary_dim": rotary_dim, "offset": offset, "sections": sections, "interleaved": interleaved, "dtype": dtype,
            "train": train, "base": base}


def _select_case(name, seqs, lo, hi, rows, hq, hkv, dims, dtype="bf16", n_sel=16, l_prime=64, empty=0):
    """`seqs` sequences of `lo` to `hi` tokens (the first `empty` of none); `rows` new ones each, n > 1 for 1 to n in turn."""
    return {"name": name, "kind": "select", "seqs": seqs, "lo": lo, "hi": hi, "rows": rows, "hq": hq, "hkv": hkv,
            "d_qk": dims[0], "d_v": dims[1], "dtype": dtype, "n_sel": n_sel, "l_prime": l_prime, "empty": empty}


def listed():
    return [
        # one decode step of a few sequences: latency
        _reserve_case("reserve_step_8", 8, 160, 1, 9000, 1, False),
        # a large decode batch in which some have ended and some wait
        _reserve_case("reserve_step_512", 512, 256, 1, 16000, 1, False, ended=0.05, idle=0.1),
        # drafted tokens of very many short sequences, odd everywhere
        _reserve_case("reserve_drafts_2999", 2999, 67, 0, 4000, 5, True, ended=0.02, idle=0.03),
        # prompts admitted at once, more than there are pages for
        _reserve_case("reserve_prompts_257", 257, 64, 0, 70, 2045, True, ended=0.1, short=0.2),
        # one decode step of a few sequences, three axes: latency
        _rotary_case("rotary_step_8", 0, 8, 64, 4, 128, 128, 0, "16,24,24", False),
        # the forward's headline prompt, three axes
        _rotary_case("rotary_prefill_64k", 1, 65536, 64, 4, 128, 128, 0, "16,24,24", False),
        # patches of an image, height and width, neighbouring pairs, a head size of no power of two
        _rotary_case("rotary_patches_odd", 3, 1369, 16, 16, 72, 72, 0, "18,18", True, "fp32", base=1e4),
        # a training step's forward and backward, the last third of wider heads turned
        _rotary_case("rotary_train_8k", 2, 8191, 64, 4, 192, 64, 128, "32", False, train=True),
        # one sequence's decode step: latency
        _select_case("select_1", 1, 65536, 65536, 1, 64, 4, (128, 128)),
        # a ragged decode batch
        _select_case("select_64", 64, 1, 32768, 1, 64, 4, (128, 128)),
        # a few drafted tokens a sequence, wide blocks, sequences that have ended
        _select_case("select_drafts", 41, 1, 20001, 4, 32, 4, (192, 128), "fp16", 8, 128, empty=3),
        # a large decode batch of long contexts
        _select_case("select_256", 256, 1, 65536, 1, 64, 4, (128, 128)),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("reserve", "rotary", "rotary", "select", "select"))
    if kind == "reserve":
        seqs = _log_int(rng, 1, 4096)
        width = _log_int(rng, 1, min(2048, (1 << 20) // seqs))
        packed = rng.random() < 0.6
        rows = _log_int(rng, 1, max(1, min(width * PAGE, (1 << 18) // seqs))) if packed else 1
        return _reserve_case("", seqs, width, 0, rng.randint(0, width * PAGE), rows, packed, rng.choice((0.0, 0.05, 0.5)),
                             rng.choice((0.0, 0.1)), rng.choice((0.0, 0.0, 0.3)))
    if kind == "rotary":
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        d = rng.choice((64, 72, 80, 128, 128, 192, 256))
        rotary_dim = rng.choice((d, d, d // 4 * 2, 36))
        offset = rng.choice((0, d - rotary_dim))
        hq, hkv = rng.choice(((64, 4), (32, 8), (16, 16), (7, 1), (28, 4)))
        pairs, axes = rotary_dim // 2, rng.choice((1, 2, 3))
        cut = [pairs // axes] * axes
        cut[-1] += pairs - sum(cut)
        train = rng.random() < 0.4
        most = 65536 * 68 * 128 * 2 // ((hq + hkv) * d * SIZES[dtype] * (2 if train else 1))
        total = _log_int(rng, 1, most)
        batch = rng.choice((1, 1, 2, 5)) if train or rng.random() < 0.5 else 0
        return _rotary_case("", batch, max(1, total // max(1, batch)), hq, hkv, d, rotary_dim, offset,
                            ",".join(map(str, cut)), rng.random() < 0.4, dtype, train, rng.choice((1e4, 1e6)))
    dims, dtype = rng.choice(DIMS), rng.choice(("bf16", "fp16"))
    hq, hkv = rng.choice(((64, 4), (32, 4), (16, 1), (16, 2), (8, 8), (48, 4), (28, 4), (32, 1), (5, 5)))
    rows = rng.choice((1, 1, 2, 4))
    seqs = _log_int(rng, 1, 512)
    most = 256 * 65536 * 4 * 128 // (hkv * dims[0] * rows)  # tokens that cost what the largest listed case does
    hi = _log_int(rng, 1024, max(1024, min(131072, most // seqs)))
    n_sel = rng.choice((1, 4, 8, 16, 16, 24, 64) if seqs > 8 else (8, 16, 24))
    return _select_case("", seqs, 1, hi, rows, hq, hkv, dims, dtype, n_sel, rng.choice((64, 64, 128, 256)),
                        rng.choice((0, 0, 1)) if seqs > 1 else 0)


def _sections(case):
    return [int(x) for x in case["sections"].split(",")]


def _lengths(case):
    """Tokens of each sequence of a select case, and the rows that each has in the call."""
    n, empty = case["seqs"], case["empty"]
    live = max(1, n - empty)
    lens = [0] * (n - live) + [case["lo"] + (case["hi"] - case["lo"]) * (i + 1) // live for i in range(live)]
    return lens, [1 + i % case["rows"] for i in range(n)]


def _completed(tokens):
    return (tokens - CMP_BLOCK) // CMP_STRIDE + 1 if tokens >= CMP_BLOCK else 0


def work(case):
    if case["kind"] == "reserve":
        held, rows = _requests(case)
        grown = [(h, r) for h, r in zip(held, rows) if r > 0 and h + r <= case["width"] * PAGE]
        pages = sum((h + r + PAGE - 1) // PAGE - (h + PAGE - 1) // PAGE for h, r in grown) * (1 - case["short"])
        pages += sum((h + PAGE - 1) // PAGE for h, r in zip(held, rows) if r < 0)
        n = sum(r for r in rows if r > 0) if case["packed"] else case["seqs"]
        return {"bytes": 20 * case["seqs"] + int(8 * pages) + 12 * n, "flops": 4 * n}
    if case["kind"] == "rotary":
        n, heads, axes = max(1, case["batch"]) * case["tokens"], case["hq"] + case["hkv"], len(_sections(case))
        times = 2 if case["train"] else 1
        return {"bytes": times * (2 * n * heads * case["d"] * SIZES[case["dtype"]] + 4 * axes * n),
                "flops": times * 3 * n * heads * case["rotary_dim"]}
    lens, rows = _lengths(case)
    held = case["hkv"] * 9 * case["d_qk"] // 16
    n, once, keys = sum(rows), 0, 0
    for length, r in zip(lens, rows):
        seen = [_completed(max(0, length - r + 1 + i)) for i in range(r)]
        once, keys = once + max(seen), keys + sum(seen)
    return {"bytes": once * held + n * case["hq"] * case["d_qk"] * 2 + 4 * n * case["hkv"] * case["n_sel"],
            "flops": 2 * keys * case["hkv"] * case["d_qk"]}


# ------------------------------------------------------------------ inputs
def _requests(case):
    """Tokens that each sequence holds and gets (those of ended ones are given back), in an order without system."""
    held, rows = [], []
    for i in range(case["seqs"]):
        x, y, z = ((i + 1) * math.sqrt(p) % 1 for p in (2, 3, 5))
        held.append(min(case["lo"] + int(x * (case["hi"] - case["lo"] + 1)), case["width"] * PAGE))
        fate = z - case["ended"]
        rows.append(-held[-1] if fate < 0 else 0 if fate < case["idle"] else 1 + int(y * case["rows"]))
    return held, rows


def _prepare_reserve(case, gen):
    n, width = case["seqs"], case["width"]
    order = torch.randperm(n, device="cuda", generator=gen)
    held, rows = (torch.tensor(x, dtype=torch.int32, device="cuda")[order] for x in _requests(case))
    # pages in an order of their own; behind a sequence's last page whatever stood there before
    have = (held + PAGE - 1) // PAGE
    want = ((held + rows + PAGE - 1) // PAGE - have).clamp(min=0)
    back = torch.where(rows < 0, have, 0).sum()
    used = int(have.sum())
    free = max(0, int(want.sum() * (1 - case["short"]) - back)) + (0 if case["short"] else 7)
    pool = torch.randperm(used + free + 57, device="cuda", generator=gen)[:used + free + 7].int()
    pages = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    pages[torch.arange(width, device="cuda") < have.unsqueeze(1)] = pool[free:free + used]
    return {"case": dict(case), "pages": pages, "held": held, "rows": rows, "pool": pool,
            "n_free": torch.tensor([free], dtype=torch.int32, device="cuda"),
            "n": int(rows.clamp(min=0).sum()) if case["packed"] else None}


def _prepare_rotary(case, gen):
    n, b, axes = case["tokens"], case["batch"], len(_sections(case))
    dtype = DTYPES[case["dtype"]]
    shape = (b, n) if b else (n,)

    def heads(h):
        return torch.randn(*shape, h, case["d"], device="cuda", generator=gen).to(dtype)

    state = {"case": dict(case), "q": heads(case["hq"]), "k": heads(case["hkv"])}
    # text (all axes alike) and images of 32 by 32 patches in turn, somewhere in a long context
    start = torch.randint(0, 100000, shape[:-1] + (1,), device="cuda", generator=gen)
    token = torch.arange(n, device="cuda").expand(shape)
    image = token // 1024 % 2 == 1
    at = token % 1024
    first = start + token - at
    grid = (first, first + at // 32, first + at % 32)
    pos = torch.stack([torch.where(image, g, start + token) for g in grid[:axes]]) if axes > 1 else (start + token).unsqueeze(0)
    state["positions"] = pos.int()
    if case["train"]:
        state["dq"], state["dk"] = (torch.randn(x.transpose(1, 2).shape, device="cuda", generator=gen).to(dtype)
                                    for x in (state["q"], state["k"]))
    if own:
        from nsa_hopper_b200 import ops

        state["plan"] = ops.rotary_plan(case["d"], rotary_dim=case["rotary_dim"], offset=case["offset"], base=case["base"],
                                        sections=_sections(case), interleaved=case["interleaved"])
        state["own_positions"] = state["positions"] if axes > 1 else state["positions"][0]
        if case["train"]:
            state["q"].requires_grad_()
            state["k"].requires_grad_()
    return state


def _quantise(x):
    """fp32 [..., d] to codes uint8 [..., d / 2] and scales uint8 [..., d / 16] (values of ordinary size)."""
    g = x.unflatten(-1, (-1, 16))
    raw = g.abs().amax(-1).clamp(min=6 * 2.0 ** -14) / torch.full_like(g[..., 0], 6.0)
    exponent = torch.frexp(raw).exponent - 1
    step = ((exponent + (127 - 3)) << 23).view(torch.float32)
    s = torch.round(raw / step) * step
    exponent = torch.frexp(s).exponent - 1
    eighths = torch.round(s / ((exponent + (127 - 3)) << 23).view(torch.float32)).int()
    y = g / s.unsqueeze(-1)
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int()
            + (a > 5.0).int() + (y < 0).int() * 8).flatten(-2)
    return (code[..., 0::2] + code[..., 1::2] * 16).to(torch.uint8), ((exponent + 14) * 8 + eighths).to(torch.uint8)


def _prepare_select(case, gen):
    lens, rows = _lengths(case)
    n, hq, hkv, d_qk, d_v = sum(rows), case["hq"], case["hkv"], case["d_qk"], case["d_v"]
    order = torch.randperm(case["seqs"], device="cuda", generator=gen)
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")[order]
    rows = torch.tensor(rows, dtype=torch.int32, device="cuda")[order]
    keys = torch.where(lens >= CMP_BLOCK, (lens - CMP_BLOCK) // CMP_STRIDE + 1, 0)
    need = (keys + PAGE - 1) // PAGE
    total, width = int(need.sum()), max(1, int(need.max()))
    pool = torch.randperm(total + 3, device="cuda", generator=gen)[:total].int()
    pages = torch.full((case["seqs"], width), -1, dtype=torch.int32, device="cuda")
    pages[torch.arange(width, device="cuda") < need.unsqueeze(1)] = pool
    cache = torch.zeros(total + 3, hkv, 36 * (d_qk + d_v), dtype=torch.uint8, device="cuda")
    # compressed keys: means of 32 keys whose channels are of unequal size and that share an offset, as a model's do
    gain = torch.exp(0.5 * torch.randn(d_qk, device="cuda", generator=gen))
    offset = 0.3 * torch.randn(hkv, 1, d_qk, device="cuda", generator=gen)
    for part in cache.split(max(1, (1 << 27) // (hkv * PAGE * d_qk))):
        k = (0.2 * torch.randn(part.shape[0], hkv, PAGE, d_qk, device="cuda", generator=gen) + offset) * gain
        codes, scales = _quantise(k)
        part[..., :36 * d_qk] = torch.cat((codes.flatten(-2), scales.flatten(-2)), -1)
    state = {"case": dict(case), "cache": cache, "pages": pages, "lens": lens, "n": n, "cu": None}
    if case["rows"] != 1:
        state["cu"] = torch.cat((torch.zeros(1, device="cuda"), rows.cumsum(0))).to(torch.int32)
    state["q"] = torch.randn(n, hq, d_qk, device="cuda", generator=gen).to(DTYPES[case["dtype"]])
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"reserve": _prepare_reserve, "rotary": _prepare_rotary, "select": _prepare_select}[case["kind"]](case, gen)


# ------------------------------------------------------------------ the plain form
def _reserve(state):
    pages, pool = state["pages"], state["pool"]
    n, width, p = pages.shape[0], pages.shape[1], pool.shape[0]
    h, r = state["held"].long().clamp(0, width * PAGE), state["rows"].long()
    want, old = h + r, (h + PAGE - 1) // PAGE
    grows = (r > 0) & (want <= width * PAGE)
    after = torch.where(grows, want, torch.where(r < 0, want.clamp(min=0), h))
    new = (after + PAGE - 1) // PAGE
    need, give = (new - old).clamp(min=0), (old - new).clamp(min=0)
    need_end, give_end = need.cumsum(0), give.cumsum(0)
    before = state["n_free"].long().clamp(0, p)
    top = (before + give_end[-1]).clamp(max=p)
    granted = grows & ((need_end <= top) | (need == 0))
    base = top - torch.where(granted, need, 0).sum()
    col = torch.arange(width, device="cuda")
    back = (col >= new.unsqueeze(1)) & (col < old.unsqueeze(1))
    at = before + (give_end - give - new).unsqueeze(1) + col
    at = torch.where(back & (at < p), at, p)  # (place p: nowhere)
    longer = torch.cat((pool, pool.new_zeros(1)))
    longer[at.flatten()] = pages.flatten()
    pool.copy_(longer[:p])
    take = granted.unsqueeze(1) & (col >= old.unsqueeze(1)) & (col < new.unsqueeze(1))
    source = base + (need_end - need - old).unsqueeze(1) + col
    pages.copy_(torch.where(take, longer[source.clamp(0, p)], pages))
    lens = torch.where(granted, want, 0)
    held = torch.where((r > 0) & ~granted, h, after)
    if state["n"] is None:
        cu, seq, pos = None, torch.arange(n, device="cuda"), lens - 1
    else:
        cu = torch.cat((r.new_zeros(1), r.clamp(min=0).cumsum(0)))
        row = torch.arange(state["n"], device="cuda")
        seq = (torch.searchsorted(cu, row, right=True) - 1).clamp(0, n - 1)
        pos = torch.where(granted[seq], lens[seq] - (cu[seq + 1] - row), -1)
    page = pages[seq, (pos // PAGE).clamp(min=0)].long()
    slot = torch.where((pos >= 0) & (page >= 0), page * PAGE + pos % PAGE, -1)
    return [lens.int(), pos.int(), slot, held.int(), base.int(), pages, pool] + ([] if cu is None else [cu.int()])


def _turn(x, cos, sin, case):
    """x [..., H, d] turned by cos and sin [..., 1, pairs]; computed in 32 bits."""
    lo, dim = case["offset"], case["rotary_dim"]
    y = x.float()
    part = y[..., lo:lo + dim]
    a, b = (part[..., 0::2], part[..., 1::2]) if case["interleaved"] else (part[..., :dim // 2], part[..., dim // 2:])
    c, s = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((c, s), -1).flatten(-2) if case["interleaved"] else torch.cat((c, s), -1)
    return torch.cat((y[..., :lo], turned, y[..., lo + dim:]), -1).to(x.dtype)


def _rotary(state):
    case, q, k = state["case"], state["q"], state["k"]
    pairs = case["rotary_dim"] // 2
    freq = torch.pow(case["base"], -torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)
    axis = torch.repeat_interleave(torch.arange(len(_sections(case)), device="cuda"),
                                   torch.tensor(_sections(case), device="cuda"), output_size=pairs)
    angle = state["positions"].double().movedim(0, -1)[..., axis] * freq
    cos, sin = torch.cos(angle).float().unsqueeze(-2), torch.sin(angle).float().unsqueeze(-2)
    if not case["batch"]:
        return [_turn(x, cos, sin, case) for x in (q, k)]
    out = [_turn(x, cos, sin, case).transpose(1, 2).contiguous() for x in (q, k)]
    if not case["train"]:
        return out
    return out + [_turn(x.transpose(1, 2), cos, -sin, case) for x in (state["dq"], state["dk"])]


def _rows(state):
    """Each row's sequence and position."""
    row = torch.arange(state["n"], device="cuda", dtype=torch.int32)
    lens, cu = state["lens"], state["cu"]
    if cu is None:
        return row.long(), lens[row.long()].long() - 1
    seq = torch.searchsorted(cu, row, right=True) - 1
    return seq, (lens[seq] - (cu[seq + 1] - row)).long()


def _select(state):
    """Scores in 64 bits: blocks are ranked by them."""
    case, cache = state["case"], state["cache"]
    hkv, d_qk, lp, n_sel = case["hkv"], case["d_qk"], case["l_prime"], case["n_sel"]
    seq, pos = _rows(state)
    width = state["pages"].shape[1]
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device="cuda")
    blocks = max(1, (case["hi"] + lp - 1) // lp)
    out = torch.full((state["n"], hkv, n_sel), -1, dtype=torch.int32, device="cuda")
    step = max(1, (1 << 28) // (hkv * width * PAGE * d_qk))
    for r in range(0, state["n"], step):
        tokens = (pos[r:r + step] + 1).clamp(min=0)
        m = tokens.shape[0]
        page = state["pages"][seq[r:r + step]].long()
        records = cache[page.clamp(min=0)][..., :36 * d_qk].transpose(1, 2)  # [rows, Hkv, W, K codes and scales]
        codes = records[..., :32 * d_qk].reshape(m, hkv, width * PAGE, d_qk // 2).int()
        scales = (records[..., 32 * d_qk:].int() << 7).to(torch.int16).view(torch.float16).float()
        value = table[torch.stack((codes % 16, codes // 16), -1).flatten(-2)]
        value = (value.unflatten(-1, (-1, 16)) * scales.reshape(m, hkv, width * PAGE, -1, 1)).flatten(-2).double()
        q = state["q"][r:r + step].double().unflatten(1, (hkv, -1)).sum(2)
        score = torch.matmul(value, q.unsqueeze(-1)).squeeze(-1)
        del codes, value
        # the block of compressed key i: that of place i among n_cmp from 0 to tokens - 1 (32 bits, rounded from 64)
        key = torch.arange(width * PAGE, device="cuda")
        n_cmp = torch.where(tokens >= CMP_BLOCK, (tokens - CMP_BLOCK) // CMP_STRIDE + 1, 0).unsqueeze(1)
        last = (tokens - 1).unsqueeze(1)
        gap = (last.float() / (n_cmp - 1).clamp(min=1).float()).double()
        place = torch.where(key < n_cmp // 2, gap * key, last.double() - gap * (n_cmp - 1 - key)).float()
        place = torch.where(n_cmp > 1, place, 0.0)
        block = (place / lp).floor().long().clamp(0, blocks - 1)
        there = (key < n_cmp) & (page.repeat_interleave(PAGE, 1) >= 0)
        total = torch.zeros(m, hkv, blocks, dtype=torch.float64, device="cuda")
        total.scatter_add_(2, block.unsqueeze(1).expand_as(score), torch.where(there.unsqueeze(1), score, 0.0))
        visible = torch.arange(blocks, device="cuda") * lp < tokens.unsqueeze(1)
        total = torch.where(visible.unsqueeze(1), total, -math.inf)
        best, index = torch.sort(total, dim=-1, descending=True, stable=True)
        k = min(n_sel, blocks)
        out[r:r + step, :, :k] = torch.where(best[..., :k] > -math.inf, index[..., :k], -1).int()
    return out


def _own(state):
    from nsa_hopper_b200 import ops

    case = state["case"]
    if case["kind"] == "reserve":
        # (the lengths are the scheduler's, which may still drop the step: `update`)
        batch = ops.cache_reserve(state["pages"], state["held"], state["rows"], state["pool"], state["n_free"],
                                  n_tokens=state["n"], update=False)
        out = [batch.lens, batch.positions, batch.slots, batch.held, batch.n_free, state["pages"], state["pool"]]
        return out if state["n"] is None else out + [batch.cu_seqlens]
    if case["kind"] == "select":
        return ops.cache_select(state["q"], state["cache"], state["pages"], state["lens"], case["n_sel"],
                                l_prime=case["l_prime"], cmp_block=CMP_BLOCK, cmp_stride=CMP_STRIDE, cu_seqlens=state["cu"])
    q, k = state["q"], state["k"]
    if case["batch"]:
        q, k = q.transpose(1, 2), k.transpose(1, 2)
    out = ops.rotary(q, k, state["own_positions"], state["plan"])
    if not case["train"]:
        return list(out)
    grads = torch.autograd.grad(out, (state["q"], state["k"]), (state["dq"], state["dk"]))
    return [x.detach() for x in out] + list(grads)


def run(state):
    if own:
        return _own(state)
    return {"reserve": _reserve, "rotary": _rotary, "select": _select}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ the definition
def _exact_reserve(state):
    """One sequence after the other, with a list as the pool."""
    pages, pool = state["pages"].cpu().numpy().copy(), state["pool"].cpu().numpy().copy()
    rows, held = state["rows"].tolist(), state["held"].tolist()
    n, width = pages.shape
    free = pool[:int(state["n_free"][0])].tolist()

    def count(tokens):
        return -(-tokens // PAGE)

    for s in range(n):
        if rows[s] < 0:
            free += pages[s, count(max(0, held[s] + rows[s])):count(held[s])].tolist()
            held[s] = max(0, held[s] + rows[s])
    pool[:len(free)] = free
    grants, wanted = [], 0
    for s in range(n):
        if rows[s] > 0 and held[s] + rows[s] <= width * PAGE:
            need = count(held[s] + rows[s]) - count(held[s])
            wanted += need
            if need == 0 or wanted <= len(free):
                grants.append((s, need))
    left = len(free) - sum(need for _, need in grants)
    at, lens = left, [0] * n
    for s, need in grants:
        have = count(held[s])
        pages[s, have:have + need] = free[at:at + need]
        at += need
        held[s] += rows[s]
        lens[s] = held[s]
    pos = []
    for s in range(n):
        for i in range(max(0, rows[s]) if state["n"] is not None else 1):
            behind = rows[s] - i if state["n"] is not None else 1
            pos.append((s, lens[s] - behind if lens[s] else -1))
    slot = [int(pages[s, t // PAGE]) * PAGE + t % PAGE if t >= 0 else -1 for s, t in pos]

    def whole(x, dtype=torch.int32):
        return torch.as_tensor(np.asarray(x), device="cuda").to(dtype)

    out = [whole(lens), whole([t for _, t in pos]), whole(slot, torch.int64), whole(held), whole([left]), whole(pages), whole(pool)]
    return out if state["n"] is None else out + [whole(np.concatenate(([0], np.cumsum(np.maximum(rows, 0)))))]


def _exact_rotary(state):
    case = state["case"]
    lo, dim, sections = case["offset"], case["rotary_dim"], _sections(case)
    pairs = dim // 2
    shift = []  # angle of every pair, one at a time
    for i in range(pairs):
        axis = sum(i >= sum(sections[:j + 1]) for j in range(len(sections)))
        shift.append(state["positions"][axis].double() * case["base"] ** (-i / pairs))
    angle = torch.stack(shift, -1).unsqueeze(-2)

    def turned(x, sign):
        out = x.detach().double()
        for a in range(0, out.shape[-2], 8):  # (some heads at a time)
            part = out[..., a:a + 8, lo:lo + dim]
            z = torch.complex(part[..., 0::2], part[..., 1::2]) if case["interleaved"] else \
                torch.complex(part[..., :pairs].contiguous(), part[..., pairs:].contiguous())
            z = z * torch.polar(torch.ones_like(angle), sign * angle)
            part.copy_(torch.view_as_real(z).flatten(-2) if case["interleaved"] else torch.cat((z.real, z.imag), -1))
        return out

    out = [turned(state[x], 1.0) for x in ("q", "k")]
    if case["batch"]:
        out = [x.transpose(1, 2) for x in out]
    if case["train"]:
        out += [turned(state[x].transpose(1, 2), -1.0) for x in ("dq", "dk")]
    return out


def _exact_select(state):
    """Sequence by sequence; places as torch gives them on the host."""
    case, q = state["case"], state["q"].double()
    hkv, d_qk, lp, n_sel = case["hkv"], case["d_qk"], case["l_prime"], case["n_sel"]
    lens = state["lens"].tolist()
    cu = list(range(state["n"] + 1)) if state["cu"] is None else state["cu"].tolist()
    out = torch.full((state["n"], hkv, n_sel), -1, dtype=torch.int32, device="cuda")
    for s, length in enumerate(lens):
        if length == 0:
            continue
        records = state["cache"][state["pages"][s, :max(1, -(-_completed(length) // PAGE))].clamp(min=0).long()].transpose(0, 1)
        codes = records[..., :32 * d_qk].reshape(hkv, -1, d_qk // 2)
        nibble = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double()
        field, two = nibble % 8, torch.floor(nibble % 8 / 2)
        size = torch.where(two == 0, field / 2, torch.where(two == 1, 1.0, torch.where(two == 2, 2.0, 4.0)) * (1 + field % 2 / 2))
        byte = records[..., 32 * d_qk:36 * d_qk].reshape(hkv, -1, d_qk // 16)
        scale = ((8 + byte % 8).double() * ((byte.long() // 8 - 18 + 1023) << 52).view(torch.float64))
        value = (torch.where(nibble >= 8, -size, size).unflatten(-1, (-1, 16)) * scale.unsqueeze(-1)).flatten(-2)
        for r in range(cu[s], cu[s + 1]):
            tokens = length - (cu[s + 1] - r) + 1
            if tokens <= 0:
                continue
            blocks, n_cmp = -(-tokens // lp), _completed(tokens)
            score = torch.zeros(hkv, blocks, dtype=torch.float64, device="cuda")
            if n_cmp:
                key = value[:, :n_cmp] @ q[r].view(hkv, -1, d_qk).sum(1).unsqueeze(-1)
                block = torch.floor(torch.linspace(0, tokens - 1, n_cmp, dtype=torch.float32) / lp).long().clamp(max=blocks - 1)
                score.index_add_(1, block.cuda(), key.squeeze(-1))
            index = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :n_sel]
            out[r, :, :index.shape[1]] = index.int()
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"reserve": _exact_reserve, "rotary": _exact_rotary, "select": _exact_select}[case["kind"]](state)
