"""The 4-bit paged KV cache on the GPU against the 64-bit oracle: what is written and read back is
compared value for value, the attention to bounds that are added up from the kernel's roundings."""
import numpy as np
import pytest
import torch

from nsa_hopper_b200 import capi, nsa, ops
from oracle import cache as oc

pytestmark = pytest.mark.gpu

DIMS = [(64, 64), (128, 128), (192, 128), (128, 64)]
DTYPES = [torch.bfloat16, torch.float16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _batch(lens, rows, num_pages, gen, width=None):
    """Page table (pages in random order, -1 behind a sequence), lens, cu_seqlens (None if rows is None)."""
    need = [(max(x, 0) + 63) // 64 for x in lens]
    width = width or max(max(need), 1)
    order = torch.randperm(num_pages, generator=gen)[:sum(need)].int()
    assert sum(need) <= num_pages
    pages = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        pages[s, :n] = order[at:at + n]
        at += n
    cu = None if rows is None else torch.tensor([0, *np.cumsum(rows)], dtype=torch.int32)
    return pages, torch.tensor(lens, dtype=torch.int32), cu


def _filled_cache(num_pages, hkv, dims, gen, dtype=torch.bfloat16):
    """Records of K and V as a model has them (uint8), by the oracle's quantiser."""
    parts = []
    for d, gain in ((dims[0], torch.exp(0.5 * torch.randn(dims[0], generator=gen))), (dims[1], torch.ones(dims[1]))):
        x = (torch.randn(num_pages, hkv, 64, d, generator=gen) * gain).to(dtype).double().numpy()
        code, byte = oc.quantise(x)
        parts += [(code[..., 0::2] + 16 * code[..., 1::2]).reshape(num_pages, hkv, -1), byte.reshape(num_pages, hkv, -1)]
    return torch.from_numpy(np.concatenate(parts, -1).astype(np.uint8))


def _cuda(*xs):
    return [None if x is None else x.cuda() for x in xs]


def _tolerances(o, lse, absolute, size, count, vmax, d_qk, out_dtype):
    """Bounds from the kernel's roundings.  u = 2^-24, half a step of fp32; a sum of n terms is counted as 2 n u of the terms'
    absolute sum (the tensor core may cut off a whole step of the largest at each addition).
    z, a score in natural units: the products are exact; 2 d u sum|q k| scale for the sum; a Q below 2^-14 of its row's largest
      is off by up to 2^-25 of that largest, which d keys' |k| multiply: no more than d u size; the products with the scale,
      with log2 e and the subtraction of the maximum: 8 u size.
    p = exp(z - m): 2^-22 (the exponential) + dz; as fp16 2^-11 more, or 2^-25 absolute below 2^-14.
    O = sum p v / sum p: 2 n u for each sum, 2^-22 for the division and weight, half a step of the output's type.
    LSE = m + ln(sum p): dz + p's error + 2 n u + 2^-22 (the logarithm) + 8 u |LSE|."""
    u = 2.0**-24
    dz = (3 * d_qk + 8) * u * size
    p = 2.0**-22 + dz
    rel = 2.0**-11 + 2 * p + 4 * count * u + 2.0**-22
    tol_o = absolute * rel[..., None] + (count * vmax)[..., None] * 2.0**-25 + np.abs(o) * torch.finfo(out_dtype).eps / 2
    if out_dtype == torch.float16:
        tol_o = tol_o + 2.0**-25
    tol_l = np.where(np.isfinite(lse), dz + p + 2 * count * u + 2.0**-22 + 8 * u * np.abs(np.where(np.isfinite(lse), lse, 0)), 0.0)
    return tol_o, tol_l


def _check(got, ref, d_qk, dtype, what=""):
    o, lse = ref[:2]
    tol_o, tol_l = _tolerances(*ref, d_qk, dtype)
    go, gl = got[0].double().cpu().numpy(), got[1].double().cpu().numpy()
    assert got[1].dtype == torch.float32
    assert np.isfinite(go).all(), what
    bad = np.abs(go - o) > tol_o
    assert not bad.any(), f"{what}: O off by {np.abs(go - o)[bad].max()} at {np.argwhere(bad)[0]}, allowed {tol_o[bad].min()}"
    assert (np.isneginf(gl) == np.isneginf(lse)).all(), what
    f = np.isfinite(lse)
    assert (np.abs(gl[f] - lse[f]) <= tol_l[f]).all(), f"{what}: LSE off by {np.abs(gl[f] - lse[f]).max()}"


# ------------------------------------------------------------------ writing and reading back
EDGE = [0.0, -0.0, 6.0, 0.25, 0.75, 1.25, -1.75, 2.5, 3.5, -5.0, 1e-6, 2.0**-18 * 6, 2.0**-17 * 9, 61440.0, 65504.0, -60000.0]


def _rows(n, hkv, d, dtype, gen):
    x = torch.randn(n, hkv, d, generator=gen) * torch.exp2(torch.randint(-18, 14, (n, hkv, d // 16), generator=gen).float()
                                                          ).repeat_interleave(16, -1)
    x[0, 0, :16] = torch.tensor(EDGE)
    if n > 2:
        x[1, 0, :16] = torch.arange(16) / 4.0          # every border between codes at scale 0.625, ties at others
        x[2, -1] = 0
    if n > 4:
        x[3, 0, 5], x[4, 0, -1] = float("nan"), float("-inf")
    if dtype == torch.bfloat16 and n > 5:
        x[5, 0, 16:32] = 3e38
    return x.to(dtype)


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,rows", [
    ([1, 64, 65, 500, 7, 130], None),
    ([70, 0, 129, 64, 1], [70, 0, 129, 64, 1]),          # whole prompts, one of them empty
    ([70, 3, 129, 200, 0], [5, 7, 64, 1, 2]),            # newest rows; more rows than tokens
])
def test_write_then_read_is_the_definition(dims, dtype, lens, rows):
    gen = _gen(1)
    hkv = 3
    pages, lens, cu = _batch(lens, rows, 24, gen)
    n = len(lens) if rows is None else sum(rows)
    k, v = _rows(n, hkv, dims[0], dtype, gen), _rows(n, hkv, dims[1], dtype, gen)
    before = torch.randint(0, 256, (24, hkv, 36 * sum(dims)), generator=gen, dtype=torch.uint8)
    cache, kd, vd, pd, ld, cd = _cuda(before, k, v, pages, lens, cu)
    assert ops.cache_write(cache, kd, vd, pd, ld, cd) is None
    after = cache.cpu().numpy()
    # bytes: the named tokens as the oracle has them, all others untouched
    want = before.numpy().copy()
    parts = oc.split(want, *dims)
    for i in range(4):
        parts[i] = parts[i].copy()
    rk, rv = np.zeros((hkv, n, dims[0])), np.zeros((hkv, n, dims[1]))
    for r in range(n):
        _, pos, page = oc.place(r, pages.numpy(), lens.numpy(), None if cu is None else cu.numpy(), 24)
        if page < 0:
            continue
        for x, c, s, back in ((k, 0, 1, rk), (v, 2, 3, rv)):
            code, byte = oc.quantise(x[r].double().numpy())
            parts[c][page, :, pos % 64] = code[..., 0::2] + 16 * code[..., 1::2]
            parts[s][page, :, pos % 64] = byte
            back[:, r] = oc.values(code, byte)
    want = np.concatenate([p.reshape(24, hkv, -1) for p in parts], -1)
    got, ref = oc.split(after, *dims), oc.split(want, *dims)
    for i in (1, 3):
        assert (got[i] == ref[i]).all()
    for i in (0, 2):
        a, b = np.stack((got[i] & 15, got[i] >> 4)), np.stack((ref[i] & 15, ref[i] >> 4))
        assert ((a == b) | ((a & 7 == 0) & (b & 7 == 0))).all()  # (the sign of a zero is free)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        a, b = ops.cache_read(cache, dims[0], pd, ld, cd, n, out)
        assert a.shape == (1, hkv, n, dims[0]) and b.shape == (1, hkv, n, dims[1]) and a.dtype == out
        for x, y in ((a, rk), (b, rv)):
            np.testing.assert_array_equal(x[0].double().cpu().numpy(), y)


def test_write_takes_strided_rows_and_pages():
    gen = _gen(2)
    hkv, dims, T = 2, (128, 64), 200
    pages, lens, cu = _batch([T], [T], 8, gen)
    kf, vf = torch.randn(1, hkv, T, 128, generator=gen).half().cuda(), torch.randn(1, hkv, T, 64, generator=gen).half().cuda()
    layers = torch.zeros(8, 3, hkv, 36 * 192, dtype=torch.uint8, device="cuda")
    plain = ops.cache_alloc(8, hkv, *dims)
    pd, ld, cd = _cuda(pages, lens, cu)
    ops.cache_write(layers[:, 1], kf[0].transpose(0, 1), vf[0].transpose(0, 1), pd, ld, cd)   # the forward's layout
    ops.cache_write(plain, kf[0].transpose(0, 1).contiguous(), vf[0].transpose(0, 1).contiguous(), pd, ld, cd)
    assert torch.equal(layers[:, 1], plain) and not layers[:, 0].any() and not layers[:, 2].any()
    both = [ops.cache_read(c, 128, pd, ld, cd, T, torch.float16) for c in (layers[:, 1], plain)]
    assert torch.equal(both[0][0], both[1][0]) and torch.equal(both[0][1], both[1][1])
    one = torch.randn(T, 1, 128, generator=gen).half().cuda()
    ops.cache_write(plain, one.expand(T, hkv, 128), vf[0].transpose(0, 1), pd, ld, cd)         # one head for all
    k, _ = ops.cache_read(plain, 128, pd, ld, cd, T)
    assert torch.equal(k[0, 0], k[0, 1])
    # a table that is a view of a wider one
    wide = torch.full((1, 9), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + pages.shape[1]] = pd
    again, _ = ops.cache_read(plain, 128, wide[:, 2:2 + pages.shape[1]], ld, cd, T)
    assert torch.equal(again, k)


@pytest.mark.parametrize("dims,hkv,lens", [((192, 128), 4, [9000, 0, 33001, 7]), ((64, 64), 2, [200001])])
def test_long_inputs_come_back(dims, hkv, lens):
    """Enough rows for the kernels' forms for long inputs, an odd number of them, and three rows of no sequence."""
    gen = _gen(4)
    n = sum(lens)
    num_pages = sum((x + 63) // 64 for x in lens)
    pages, lens, cu = _batch(lens, lens, num_pages, gen)
    k, v = torch.randn(n + 3, hkv, dims[0], generator=gen).bfloat16(), torch.randn(n + 3, hkv, dims[1], generator=gen).bfloat16()
    cache = ops.cache_alloc(num_pages, hkv, *dims)
    kd, vd, pd, ld, cd = _cuda(k, v, pages, lens, cu)
    ops.cache_write(cache, kd, vd, pd, ld, cd)
    for dtype in (torch.bfloat16, torch.float32):
        for x, y in zip(ops.cache_read(cache, dims[0], pd, ld, cd, n + 3, dtype), (k, v)):
            assert not x[0, :, n:].any()
            at = torch.cat((torch.arange(0, n, 997), torch.arange(n - 130, n)))
            np.testing.assert_array_equal(x[0, :, :n].cpu()[:, at].double().numpy().transpose(1, 0, 2),
                                          oc.values(*oc.quantise(y[at].double().numpy())))


def test_absent_tokens_are_skipped():
    """Pages outside the cache, lengths behind the table, negative lengths, rows of no sequence."""
    gen = _gen(3)
    hkv, dims, P = 2, (64, 64), 4
    pages = torch.tensor([[0, -1, 9, 1], [2, 3, -2**31, 2**31 - 1], [0, 1, 2, 3]], dtype=torch.int32)
    lens = torch.tensor([256, 2**31 - 1, -5], dtype=torch.int32)
    cu = torch.tensor([2, 258, 300, 310], dtype=torch.int32)
    n = 320
    k, v = torch.randn(n, hkv, 64, generator=gen).bfloat16(), torch.randn(n, hkv, 64, generator=gen).bfloat16()
    before = torch.full((P, hkv, 36 * 128), 0x11, dtype=torch.uint8)
    cache, kd, vd, pd, ld, cd = _cuda(before, k, v, pages, lens, cu)
    ops.cache_write(cache, kd, vd, pd, ld, cd)
    got = cache.cpu()
    assert torch.equal(got[2:], before[2:]) and not (got[:2] == before[:2]).all()
    kr, vr = ops.cache_read(cache, 64, pd, ld, cd, n, torch.float32)
    there = torch.zeros(n, dtype=torch.bool)
    there[2:66] = there[194:258] = True
    assert not kr[0][:, ~there].any() and not vr[0][:, ~there].any()
    np.testing.assert_array_equal(kr[0][:, there].cpu().numpy(),
                                  oc.values(*oc.quantise(k.double().numpy())).transpose(1, 0, 2)[:, there.numpy()])
    q = torch.randn(n, 4, 64, generator=gen).bfloat16()
    for window, sel in ((0, None), (100, None), (0, torch.randint(-2, 6, (n, hkv, 5), generator=gen, dtype=torch.int32))):
        got = ops.cache_attend(q.cuda(), cache, pd, ld, sel=None if sel is None else sel.cuda(), window=window, cu_seqlens=cd)
        ref = oc.attend(q.double().numpy(), cache.cpu().numpy(), pages.numpy(), lens.numpy(),
                        None if sel is None else sel.numpy(), window=window, cu=cu.numpy())
        _check(got, ref, 64, torch.bfloat16)


def test_empty_calls():
    cache = ops.cache_alloc(2, 2, 128, 128)
    e = torch.empty
    pages, lens = e(0, 3, dtype=torch.int32, device="cuda"), e(0, dtype=torch.int32, device="cuda")
    k = e(0, 2, 128, dtype=torch.bfloat16, device="cuda")
    ops.cache_write(cache, k, k, pages, lens)
    assert ops.cache_read(cache, 128, pages, lens)[0].shape == (1, 2, 0, 128)
    o, lse = ops.cache_attend(e(0, 8, 128, dtype=torch.bfloat16, device="cuda"), cache, pages, lens)
    assert o.shape == (0, 8, 128) and lse.shape == (0, 8)
    # sequences without a page, a cache without pages
    pages, lens = e(3, 0, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    for c in (cache, ops.cache_alloc(0, 2, 128, 128)):
        o, lse = ops.cache_attend(torch.ones(3, 8, 128, dtype=torch.bfloat16, device="cuda"), c, pages, lens)
        assert not o.any() and torch.isneginf(lse).all()


# ------------------------------------------------------------------ attention
def _attend_case(dims, hq, hkv, lens, rows, dtype, seed, *, n_sel=0, l_prime=64, window=0, scale=0.0, tail=0, poison=True):
    gen = _gen(seed)
    num_pages = sum((max(x, 0) + 63) // 64 for x in lens) + 2
    pages, lens, cu = _batch(lens, rows, num_pages, gen)
    cache = _filled_cache(num_pages, hkv, dims, gen)
    if poison:  # behind every sequence's last token, and in pages of nobody: scales that are NaN
        parts = [p.clone() for p in map(torch.from_numpy, oc.split(cache.numpy(), *dims))]
        owner = {int(p): (s, i) for s in range(len(lens)) for i, p in enumerate(pages[s].tolist()) if p >= 0}
        for p in range(num_pages):
            s, i = owner.get(p, (0, 10**6))
            first = max(0, min(64, int(lens[s]) - 64 * i)) if p in owner else 0
            for part in parts:
                part[p, :, first:] = 0xFF
        cache = torch.cat([p.reshape(num_pages, hkv, -1) for p in parts], -1)
    n = (len(lens) if rows is None else sum(rows)) + tail
    q = torch.randn(n, hq, dims[0], generator=gen).to(dtype)
    sel = None
    if n_sel:
        top = max(int(lens.max()) // l_prime + 2, 2)
        sel = torch.randint(-1, top, (n, hkv, n_sel), generator=gen, dtype=torch.int32)  # duplicates, padding, future blocks
    qd, cd, pd, ld, cud, sd = _cuda(q, cache, pages, lens, cu, sel)
    got = ops.cache_attend(qd, cd, pd, ld, sel=sd, l_prime=l_prime, window=window, cu_seqlens=cud, scale=scale)
    assert got[0].dtype == dtype and got[0].shape == (n, hq, dims[1])
    ref = oc.attend(q.double().numpy(), cache.numpy(), pages.numpy(), lens.numpy(), None if sel is None else sel.numpy(), l_prime,
                    window, None if cu is None else cu.numpy(), scale)
    _check(got, ref, dims[0], dtype, f"{dims} {hq}/{hkv} n_sel={n_sel} window={window}")
    return got


LENS = [0, 1, 2, 63, 64, 65, 127, 128, 129, 300, 1000]


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mode", [dict(), dict(n_sel=4), dict(n_sel=3, l_prime=256), dict(window=1), dict(window=70),
                                  dict(window=100, n_sel=6), dict(window=2**31 - 1)])
def test_attend(dims, dtype, mode):
    _attend_case(dims, 32, 2, LENS, None, dtype, 5, **mode)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (5, 5), (8, 2), (15, 3), (17, 1), (32, 1), (48, 2), (128, 1)])
@pytest.mark.parametrize("mode", [dict(), dict(n_sel=5, l_prime=128)])
def test_attend_groups(hq, hkv, mode):
    _attend_case((128, 128), hq, hkv, [130, 1, 700], None, torch.bfloat16, 6, **mode)


@pytest.mark.parametrize("rows", [[1, 0, 3, 4, 2], [5, 1, 0, 0, 3]])
@pytest.mark.parametrize("mode", [dict(), dict(n_sel=4), dict(window=65)])
def test_attend_several_rows_a_sequence(rows, mode):
    _attend_case((128, 128), 16, 2, [64, 3, 2, 513, 129], rows, torch.float16, 7, tail=3, **mode)


@pytest.mark.parametrize("n_sel,l_prime", [(33, 64), (40, 128), (1, 256), (129, 64), (1024, 64)])
def test_attend_long_selections(n_sel, l_prime):
    _attend_case((64, 64), 8, 2, [3000, 900], None, torch.bfloat16, 8, n_sel=n_sel, l_prime=l_prime)


def _random_cache(num_pages, hkv, dims, gen):
    """Records of random codes, with scales between 0.04 and 0.6."""
    parts = []
    for d in dims:
        parts.append(torch.randint(0, 256, (num_pages, hkv, 32 * d), generator=gen, dtype=torch.uint8))
        parts.append(torch.randint(0x52, 0x72, (num_pages, hkv, 4 * d), generator=gen, dtype=torch.uint8))
    return torch.cat(parts, -1)


def _plan(n, hq, hkv, dims, width, n_sel, l_prime, window):
    batch = capi.make_cache_batch(cache=256, pages=256, lens=256, num_pages=1, n_seqs=n, width=width, n_rows=n, heads_kv=hkv,
                                  d_qk=dims[0], d_v=dims[1])
    return capi.cache_attend_plan(capi.make_cache_attend_desc(batch=batch, q=256, o=256, heads_q=hq, sel=256 if n_sel else 0,
                                                              n_sel=n_sel, block_size=l_prime, window=window), 0)


# lengths, width of the page table, selection, head dims, heads; what the plan has to be for the case to be what it stands for
SHARING = [
    ([2100], 33, 0, (128, 128), (16, 1), dict(cluster=8, merge=0)),
    ([2100, 3, 0, 64], 33, 0, (64, 64), (4, 1), dict(cluster=8, merge=0)),
    ([1500] * 6, 24, 0, (128, 128), (24, 4), dict(cluster=4, merge=0)),
    ([700, 1, 650], 16, 9, (192, 128), (64, 8), dict(cluster=2, merge=0)),
    ([900] * 30, 40, 16, (128, 64), (8, 4), dict(cluster=1, team=8, merge=0)),
    ([500] * 60, 8, 16, (128, 128), (32, 4), dict(cluster=1, team=4, merge=0)),
    ([900] * 120, 16, 16, (64, 64), (32, 4), dict(cluster=1, team=2, merge=0)),
    ([300] * 600, 6, 3, (64, 64), (4, 2), dict(cluster=1, team=1, merge=0)),
    ([130, 70, 0, 200] * 500, 60, 0, (64, 64), (2, 1), dict(slots=60, cluster=1)),    # more rows than a ragged line takes
    ([130, 70, 0, 6000] + [200] * 2000, 900, 0, (64, 64), (2, 1), dict(slots=900, cluster=1)),  # and a wide table
    ([25000], 391, 0, (128, 128), (16, 1), dict(slots=0, merge=8)),                   # cut, eight warps join
    ([20000, 1, 0, 64, 9999], 2000, 0, (192, 128), (6, 2), dict(slots=0, merge=8)),
    ([5000] * 40 + [0, 1, 64], 200, 0, (128, 64), (48, 1), dict(slots=0, merge=1)),   # cut, one warp joins
    ([30000] * 20 + [1] * 20, 480, 0, (64, 64), (8, 2), dict(slots=0)),               # long enough for warps of their own
    ([40000] * 2, 630, 600, (64, 64), (17, 1), dict(slots=600, merge=8)),             # long selections are cut, too
]


@pytest.mark.parametrize("lens,width,n_sel,dims,heads,want", SHARING, ids=[str(i) for i in range(len(SHARING))])
def test_attend_however_the_work_is_shared(lens, width, n_sel, dims, heads, want):
    (hq, hkv), n = heads, len(lens)
    plan = _plan(n, hq, hkv, dims, width, n_sel, 64, 0)
    assert {k: plan[k] for k in want} == want
    gen = _gen(40 + n)
    num_pages = sum((x + 63) // 64 for x in lens)
    pages, lens, _ = _batch(lens, None, num_pages, gen, width)
    cache = _random_cache(num_pages, hkv, dims, gen)
    q = torch.randn(n, hq, dims[0], generator=gen).bfloat16()
    sel = None
    if n_sel:
        sel = torch.randint(-1, width, (n, hkv, n_sel), generator=gen, dtype=torch.int32)
        sel[:, :, 0] = torch.clamp(lens - 1, min=0).view(-1, 1) // 64
    args = _cuda(q, cache, pages, lens)
    got = ops.cache_attend(*args, sel=None if sel is None else sel.cuda())
    ref = oc.attend(q.double().numpy(), cache.numpy(), pages.numpy(), lens.numpy(), None if sel is None else sel.numpy())
    _check(got, ref, dims[0], torch.bfloat16)
    again = ops.cache_attend(*args, sel=None if sel is None else sel.cuda())
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    # the same rows through `out`, with cu_seqlens, and one row of no sequence behind, which stays
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    q1 = torch.cat((args[0], args[0][:1]))
    s1 = None if sel is None else torch.cat((sel, sel[:1])).cuda()
    out = torch.full((n + 1, hq, dims[1]), 3.0, device="cuda")
    o, lse = ops.cache_attend(q1, *args[1:], sel=s1, cu_seqlens=cu, out=out, accumulate=True)
    assert (o[n] == 3).all() and torch.isneginf(lse[n]).all()
    tol = _tolerances(*ref, dims[0], torch.float32)[0]
    assert (np.abs(o[:n].double().cpu().numpy() - 3 - ref[0]) <= tol + 2.0**-21).all()


@pytest.mark.parametrize("seed", range(40))
def test_attend_random_calls(seed):
    """Shapes, tables and lengths at random, broken ones among them."""
    rng = np.random.default_rng(100 + seed)
    gen = _gen(100 + seed)
    dims, dtype = DIMS[rng.integers(4)], DTYPES[rng.integers(2)]
    hkv = int(rng.integers(1, 5))
    hq = hkv * int(rng.choice([1, 3, 8, 9, 16, 20]))
    S, width, P = int(rng.integers(1, 12)), int(rng.integers(1, 24)), 64
    lens = np.where(rng.random(S) < 0.2, rng.choice([0, -3, width * 64, width * 64 + 5]), rng.integers(1, width * 64 + 1, S))
    pages = rng.permutation(np.tile(np.arange(P), S * width // P + 1))[:S * width].reshape(S, width).astype(np.int32)
    pages[rng.random((S, width)) < 0.1] = rng.choice([-1, P, P + 7, -2**31])
    rows = None if rng.random() < 0.4 else rng.integers(0, 5, S)
    n = S if rows is None else int(rows.sum()) + int(rng.integers(0, 3))
    cu = None if rows is None else np.concatenate(([0], rows.cumsum())).astype(np.int32)
    n = max(n, 1) if rows is not None else n
    n_sel = int(rng.choice([0, 0, 1, 7, 40]))
    l_prime = int(rng.choice([64, 128, 256]))
    window = int(rng.choice([0, 0, 1, 63, 200, 5000]))
    cache = _random_cache(P, hkv, dims, gen)
    q = torch.randn(n, hq, dims[0], generator=gen).to(dtype)
    sel = rng.integers(-2, width * 64 // l_prime + 2, (n, hkv, n_sel)).astype(np.int32) if n_sel else None
    t = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    lens = lens.astype(np.int32)
    got = ops.cache_attend(q.cuda(), cache.cuda(), t(pages), t(lens), sel=t(sel), l_prime=l_prime, window=window, cu_seqlens=t(cu))
    ref = oc.attend(q.double().numpy(), cache.numpy(), pages, lens, sel, l_prime, window, cu)
    _check(got, ref, dims[0], dtype, f"seed {seed}")


def test_attend_scale_and_large_queries():
    _attend_case((128, 128), 16, 1, [500], None, torch.bfloat16, 13, scale=0.7)
    gen = _gen(14)
    dims, hkv = (128, 128), 1
    pages, lens, _ = _batch([200, 200, 200, 200], None, 16, gen)
    cache = _filled_cache(16, hkv, dims, gen)
    q = torch.randn(4, 16, 128, generator=gen)
    q[0] *= 2.0**100   # far outside fp16: the row's power of two
    q[1] *= 2.0**-100
    q[2, :, ::2] *= 2.0**-20  # small values beside large ones
    q[3] = 0
    q = q.bfloat16()
    scale = 2.0**-100
    for rows, sc in ((slice(0, 1), scale), (slice(1, 4), 0.0)):
        qd, cd, pd, ld = _cuda(q[rows], cache, pages[rows], lens[rows])
        got = ops.cache_attend(qd.contiguous(), cd, pd.contiguous(), ld.contiguous(), scale=sc)
        _check(got, oc.attend(q[rows].double().numpy(), cache.numpy(), pages[rows].numpy(), lens[rows].numpy(), scale=sc), 128,
               torch.bfloat16)


def test_attend_nan_and_infinity_in_visible_places_come_through():
    gen = _gen(15)
    pages, lens, _ = _batch([100, 100, 100], None, 8, gen)
    cache, pd, ld = _cuda(ops.cache_alloc(8, 1, 128, 128, "cpu"), pages, lens)
    k, v = torch.randn(300, 1, 128, generator=gen), torch.randn(300, 1, 128, generator=gen)
    k[30, 0, 5] = float("nan")     # sequence 0: a key
    v[130, 0, 40] = float("inf")   # sequence 1: a value: its group of 16
    cu = torch.tensor([0, 100, 200, 300], dtype=torch.int32, device="cuda")
    ops.cache_write(cache, k.bfloat16().cuda(), v.bfloat16().cuda(), pd, ld, cu)
    q = torch.randn(3, 4, 128, generator=gen).bfloat16().cuda()
    o, lse = ops.cache_attend(q, cache, pd, ld)
    assert o[0].isnan().all() and lse[0].isnan().all()
    assert o[1, :, 32:48].isnan().all() and o[1, :, :32].isfinite().all() and o[1, :, 48:].isfinite().all() and lse[1].isfinite().all()
    assert o[2].isfinite().all()
    # before the window, or in a block that is not selected, they are not met
    o, lse = ops.cache_attend(q, cache, pd, ld, window=69)
    assert o.isfinite().all() and lse.isfinite().all()
    sel = torch.ones(3, 1, 1, dtype=torch.int32, device="cuda")
    assert ops.cache_attend(q, cache, pd, ld, sel=sel)[0].isfinite().all()


def test_attend_out_weight_accumulate():
    gen = _gen(16)
    hkv, dims = 2, (128, 128)
    pages, lens, cu = _batch([300, 0, 70], [2, 1, 2], 8, gen)
    cache = _filled_cache(8, hkv, dims, gen)
    q = torch.randn(7, 16, 128, generator=gen).bfloat16()  # two rows behind the last sequence
    qd, cd, pd, ld, cud = _cuda(q, cache, pages, lens, cu)
    base = torch.randn(7, 16, 128, generator=gen).cuda()
    w = torch.tensor([0.75, 9.0], device="cuda")
    ref = oc.attend(q.double().numpy(), cache.numpy(), pages.numpy(), lens.numpy(), cu=cu.numpy())
    tol = _tolerances(*ref, 128, torch.float32)[0]
    for accumulate in (False, True):
        out = base.clone()
        o, lse = ops.cache_attend(qd, cd, pd, ld, cu_seqlens=cud, out=out, weight=w, accumulate=accumulate)
        assert o.data_ptr() == out.data_ptr()
        want = ref[0] * 0.75 + (base.double().cpu().numpy() if accumulate else 0)
        got = out.double().cpu().numpy()
        assert (np.abs(got - want)[:5] <= tol[:5] + np.abs(want[:5]) * 2.0**-23).all()
        assert torch.equal(out[5:], base[5:]) and torch.isneginf(lse[5:]).all() and torch.isneginf(lse[2]).all()
    o, lse = ops.cache_attend(qd, cd, pd, ld, cu_seqlens=cud)
    assert not o[5:].any() and torch.isneginf(lse[5:]).all()
    assert ops.cache_attend(qd, cd, pd, ld, cu_seqlens=cud, with_lse=False)[1].numel() == 0
    out = torch.empty(7, 16, 128, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(ops.cache_attend(qd, cd, pd, ld, cu_seqlens=cud, out=out)[0][:5], o[:5])


def test_attend_strided_queries():
    gen = _gen(17)
    pages, lens, _ = _batch([300, 65], None, 8, gen)
    cache = _filled_cache(8, 2, (64, 64), gen)
    cd, pd, ld = _cuda(cache, pages, lens)
    qkv = torch.randn(2, 3, 8, 64, generator=gen).bfloat16().cuda()
    want = ops.cache_attend(qkv[:, 1].contiguous(), cd, pd, ld)
    for q in (qkv[:, 1], qkv[:, 1].transpose(0, 1).contiguous().transpose(0, 1)):
        got = ops.cache_attend(q, cd, pd, ld)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = qkv[:, 1, :1]
    got = ops.cache_attend(one.expand(2, 8, 64), cd, pd, ld)
    assert torch.equal(got[0], ops.cache_attend(one.expand(2, 8, 64).contiguous(), cd, pd, ld)[0])


def test_refusals_on_the_device():
    cache = ops.cache_alloc(4, 2, 128, 128)
    i32 = dict(dtype=torch.int32, device="cuda")
    pages, lens = torch.zeros(3, 2, **i32), torch.ones(3, **i32)
    q = torch.zeros(3, 8, 128, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device="cuda")
    for bad, match in (
            (lambda: ops.cache_attend(q[:, :7], cache, pages, lens), "multiple of Hkv"),
            (lambda: ops.cache_attend(q, cache, pages.long(), lens), "int32"),
            (lambda: ops.cache_attend(q, cache, pages[:2], lens), "one row for each sequence"),
            (lambda: ops.cache_attend(q[:2], cache, pages, lens), "one row for each sequence"),
            (lambda: ops.cache_attend(q[..., :64], cache, pages, lens), "not one of"),
            (lambda: ops.cache_attend(q, cache[..., :9200], pages, lens), "not one of|record"),
            (lambda: ops.cache_attend(q, cache, pages, lens, sel=torch.zeros(3, 1, 4, **i32)), "sel must be"),
            (lambda: ops.cache_attend(q, cache, pages, lens, sel=torch.zeros(3, 2, 4, **i32), l_prime=96), "block_size"),
            (lambda: ops.cache_attend(q, cache, pages, lens, window=-1), "negative"),
            (lambda: ops.cache_attend(q, cache, pages, lens, accumulate=True), "needs an out"),
            (lambda: ops.cache_attend(q, cache, pages, lens, out=torch.empty_like(q), accumulate=True), "fp32 out"),
            (lambda: ops.cache_attend(q, cache, pages, lens, out=torch.empty(3, 8, 64, device="cuda")), "out must be"),
            (lambda: ops.cache_attend(q, cache, pages, lens.cpu()), "device"),
            (lambda: ops.cache_attend(q, cache, pages, lens, cu_seqlens=lens), "one entry more"),
            (lambda: ops.cache_write(cache, k[:, :1], k[:, :1], pages, lens), "same heads"),
            (lambda: ops.cache_write(cache, k, k[..., 1:], pages, lens), "not one of"),
            (lambda: ops.cache_write(cache, torch.zeros(3, 2, 132, dtype=torch.bfloat16, device="cuda")[..., :128], k, pages, lens),
             "multiples of 8"),
            (lambda: ops.cache_write(cache, k.float(), k.float(), pages, lens), "bfloat16 or float16"),
            (lambda: ops.cache_read(cache, 96, pages, lens), "not one of"),
            (lambda: ops.cache_read(cache, 128, pages, lens, dtype=torch.int8), "dtype must be"),
            (lambda: ops.cache_read(cache, 128, pages, lens, n_tokens=2), "one row for each sequence"),
    ):
        with pytest.raises(RuntimeError, match=match):
            bad()


# ------------------------------------------------------------------ streams, graphs, large caches, order
def _small(seed, n=3, hq=16, hkv=2):
    gen = _gen(seed)
    pages, lens, _ = _batch([500, 64, 3000][:n], None, 64, gen)
    return [x.cuda() for x in (torch.randn(n, hq, 128, generator=gen).bfloat16(), _filled_cache(64, hkv, (128, 128), gen), pages, lens)]


def test_attend_repeats_to_the_bit():
    q, cache, pages, lens = _small(20)
    first = ops.cache_attend(q, cache, pages, lens)
    for _ in range(5):
        again = ops.cache_attend(q, cache, pages, lens)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_two_graphs_and_eager_calls_at_once():
    """A captured decode step (write, attend) replayed on new contents, beside another graph and eager calls."""
    q, cache, pages, lens = _small(21)
    k = torch.randn(3, 2, 128, device="cuda").bfloat16()
    want0 = ops.cache_attend(q, cache, pages, lens)
    streams = [torch.cuda.Stream() for _ in range(3)]
    graphs, outs, queries = [], [], []
    for s in streams[:2]:
        x = q.clone()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(ops.cache_attend(x, cache, pages, lens))
        graphs.append(g)
        queries.append(x)
    queries[1].mul_(-1)
    want1 = ops.cache_attend(-q, cache, pages, lens)
    torch.cuda.synchronize()
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = ops.cache_attend(q, cache, pages, lens)
    torch.cuda.synchronize()
    for got, want in ((outs[0], want0), (outs[1], want1), (eager, want0)):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # a step: the new token is written, then seen
    c2, l2 = cache.clone(), lens.clone()
    pages2 = pages.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.cache_write(c2, k, k, pages2, l2)
        o, _ = ops.cache_attend(q, c2, pages2, l2)
    c2.copy_(cache)
    free = [p for p in range(64) if p not in pages.tolist()[0] + pages.tolist()[1] + pages.tolist()[2]]
    for i in range(3):
        l2 += 1
        need = ((l2 + 63) // 64).tolist()
        for s in range(3):
            if need[s] <= pages2.shape[1] and int(pages2[s, need[s] - 1]) < 0:
                pages2[s, need[s] - 1] = free.pop()
        k.normal_()
        g.replay()
        torch.cuda.synchronize()
        ref = oc.attend(q.double().cpu().numpy(), c2.cpu().numpy(), pages2.cpu().numpy(), l2.cpu().numpy())
        _check((o, torch.from_numpy(ref[1]).float()), ref, 128, torch.bfloat16)
        back, _ = ops.cache_read(c2, 128, pages2, l2)
        np.testing.assert_array_equal(back[0].double().cpu().numpy().transpose(1, 0, 2),
                                      oc.values(*oc.quantise(k.double().cpu().numpy())))


@pytest.mark.parametrize("n", [1, 3])
def test_waits_are_bounded(n):
    """A launch whose copies never come ends by itself: the error word is set, the rows are NaN, the next call is right."""
    q, cache, pages, lens = _small(24, n)
    want = ops.cache_attend(q, cache, pages, lens)
    o, lse, err = torch.zeros_like(want[0]), torch.zeros_like(want[1]), torch.zeros(1, dtype=torch.int32, device="cuda")
    batch = capi.make_cache_batch(cache=cache.data_ptr(), pages=pages.data_ptr(), lens=lens.data_ptr(), num_pages=64, n_seqs=n,
                                  width=pages.shape[1], n_rows=n, heads_kv=2, d_qk=128, d_v=128)
    desc = capi.make_cache_attend_desc(batch=batch, q=q.data_ptr(), o=o.data_ptr(), lse=lse.data_ptr(), heads_q=16,
                                       err=err.data_ptr(), timeout_ms=20, debug_flags=capi.NSA_DEBUG_STALL)
    work = torch.empty(capi.cache_attend_workspace_bytes(desc), dtype=torch.uint8, device="cuda")
    desc.workspace = work.data_ptr()
    stream = torch.cuda.current_stream().cuda_stream
    capi.cache_attend(desc, stream)
    assert err.item() == capi.NSA_DEVERR_TIMEOUT and o.isnan().all() and lse.isnan().all()
    err.zero_()
    desc.debug_flags = 0
    capi.cache_attend(desc, stream)
    assert err.item() == 0 and torch.equal(o, want[0]) and torch.equal(lse, want[1])


def test_calls_in_a_row_keep_their_order():
    """The kernels are launched before the ones ahead of them end; each must still see what those wrote, and write nothing
    that they still read: a token overwritten and attended to a hundred times, without and with a wait after each call."""
    q, cache, pages, lens = _small(25)
    lens = torch.tensor([500, 64, 2100], dtype=torch.int32, device="cuda")
    ks = torch.randn(100, 3, 2, 128, device="cuda").bfloat16()
    results = []
    for wait in (True, False):
        c, outs = cache.clone(), []
        x = torch.zeros_like(ks[0])
        for k in ks:
            x.copy_(k)                                   # (a copy, then a kernel of torch's, ahead of the first)
            ops.cache_write(c, x, x.mul(2), pages, lens)
            if wait:
                torch.cuda.synchronize()
            outs += ops.cache_attend(q, c, pages, lens)
            if wait:
                torch.cuda.synchronize()
            outs += ops.cache_read(c, 128, pages, lens)
            if wait:
                torch.cuda.synchronize()
        results.append(outs)
    torch.cuda.synchronize()
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_captured_behind_copies_and_other_streams():
    q, cache, pages, lens = _small(26)
    k = torch.randn(3, 2, 128, device="cuda").bfloat16()
    c, x, l2 = cache.clone(), torch.zeros_like(q), lens.clone()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    buf = torch.empty(3, 16, 128, device="cuda")
    with torch.cuda.graph(g):
        x.copy_(q)                       # a copy node
        c.copy_(cache)
        buf.zero_()                      # a memset node
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            o1, _ = ops.cache_attend(x, c, pages, l2, window=100)
        ops.cache_attend(x, c, pages, l2, out=buf, accumulate=True)
        main.wait_stream(side)           # two nodes ahead of the next
        ops.cache_write(c, k, k, pages, l2)
        o2, _ = ops.cache_attend(x, c, pages, l2)
    for _ in range(3):
        q.mul_(-1.5)
        g.replay()
        torch.cuda.synchronize()
        fresh = cache.clone()
        assert torch.equal(o1, ops.cache_attend(q, fresh, pages, lens, window=100)[0])
        assert torch.equal(buf, ops.cache_attend(q, fresh, pages, lens, out=torch.zeros_like(buf), accumulate=True)[0])
        ops.cache_write(fresh, k, k, pages, lens)
        assert torch.equal(o2, ops.cache_attend(q, fresh, pages, lens)[0])


def test_side_stream():
    q, cache, pages, lens = _small(22)
    want = ops.cache_attend(q, cache, pages, lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x = torch.zeros_like(q)
        torch.cuda._sleep(20_000_000)
        x.copy_(q)
        got = ops.cache_attend(x, cache, pages, lens)
    s.synchronize()
    assert torch.equal(got[0], want[0])


def test_cache_beyond_32_bit_offsets():
    hkv, dims = 4, (192, 128)
    record = 36 * 320
    P = (5 << 30) // (hkv * record)
    cache = torch.empty(P, hkv, record, dtype=torch.uint8, device="cuda")
    gen = _gen(23)
    lens = torch.tensor([150, 70], dtype=torch.int32)
    pages = torch.tensor([[P - 1, 3, P - 2], [P - 5, P // 2 + 7, -1]], dtype=torch.int32)
    cu = torch.tensor([0, 150, 220], dtype=torch.int32)
    k, v = torch.randn(220, hkv, 192, generator=gen).bfloat16(), torch.randn(220, hkv, 128, generator=gen).bfloat16()
    q = torch.randn(2, 16, 192, generator=gen).bfloat16()
    kd, vd, pd, ld, cd, qd = _cuda(k, v, pages, lens, cu, q)
    ops.cache_write(cache, kd, vd, pd, ld, cd)
    kr, vr = ops.cache_read(cache, 192, pd, ld, cd, 220, torch.float32)
    np.testing.assert_array_equal(kr[0].cpu().numpy().transpose(1, 0, 2), oc.values(*oc.quantise(k.double().numpy())))
    np.testing.assert_array_equal(vr[0].cpu().numpy().transpose(1, 0, 2), oc.values(*oc.quantise(v.double().numpy())))
    got = ops.cache_attend(qd, cache, pd, ld)
    small = cache[pages.clamp(min=0).flatten().long()].cpu().numpy()
    ref = oc.attend(q.double().numpy(), small, np.where(pages.numpy() >= 0, np.arange(6).reshape(2, 3), -1), lens.numpy())
    _check(got, ref, 192, torch.bfloat16)


# ------------------------------------------------------------------ a run of them together
def test_decode_continues_a_prefill():
    """A prompt is written, its selected branch runs on what the cache holds, then tokens are decoded one by one
    through the three branches, and each is compared with the formulas on the cache's contents."""
    gen = _gen(30)
    hq, hkv, d, T0, steps, S = 16, 2, 128, 300, 20, 2
    P, W = 24, 6
    cache, cmp_cache = ops.cache_alloc(P, hkv, d, d), ops.cache_alloc(8, hkv, d, d)
    pages = torch.randperm(P, generator=gen)[:S * W].view(S, W).int().cuda()
    cmp_pages = torch.tensor([[3, 1], [0, 6]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([T0, T0 - 77], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, T0, 2 * T0 - 77], dtype=torch.int32, device="cuda")
    n = 2 * T0 - 77
    k, v = (torch.randn(n, hkv, d, generator=gen).bfloat16().cuda() for _ in range(2))
    ops.cache_write(cache, k, v, pages, lens, cu)
    K, V = ops.cache_read(cache, d, pages, lens, cu, n)
    # the prompt's last tokens: the varlen forward on the values read back, and the decode form on the cache
    q = torch.randn(1, hq, n, d, generator=gen).bfloat16().cuda()
    sel = torch.randint(0, 4, (1, hkv, n, 3), generator=gen, dtype=torch.int32).cuda()
    o1, l1 = ops.forward_lse(q, K, V, sel, 64, 1, cu_seqlens=cu, out_f32=True)
    last = (cu[1:] - 1).long()
    o2, l2 = ops.cache_attend(q[0].transpose(0, 1)[last].contiguous(), cache, pages, lens, sel=sel[0].transpose(0, 1)[last].contiguous())
    # (both round P: bf16 there, 2^-9 of each term at most, fp16 here; the output is bf16 here)
    assert (o1[0].transpose(0, 1)[last] - o2.float()).abs().max() <= (2**-8 + 2**-8 + 2**-10) * float(V.abs().max())
    assert (l1[0].transpose(0, 1)[last] - l2).abs().max() <= 1e-4
    # compressed keys of the prompt, one sequence at a time
    for s in range(S):
        Ks, Vs = (x[:, :, int(cu[s]):int(cu[s + 1])] for x in (K, V))
        kc, vc = (x[0].transpose(0, 1).bfloat16().contiguous() for x in nsa.compress_kv(Ks, Vs))
        m = kc.shape[0]
        ops.cache_write(cmp_cache, kc, vc, cmp_pages[s:s + 1].contiguous(), torch.tensor([m], dtype=torch.int32, device="cuda"),
                        torch.tensor([0, m], dtype=torch.int32, device="cuda"))
    gate_w = torch.tensor([0.3, -0.2, 0.9])
    g = nsa.gate_weights(gate_w, "cpu").double().numpy()
    for _ in range(steps):
        lens = lens + 1
        kn, vn = (torch.randn(S, hkv, d, generator=gen).bfloat16().cuda() for _ in range(2))
        ops.cache_write(cache, kn, vn, pages, lens)
        cmp_lens = nsa.cache_compress(cache, d, pages, lens, cmp_cache, cmp_pages)
        assert cmp_lens.tolist() == [(x - 32) // 16 + 1 for x in lens.tolist()]
        qn = torch.randn(S, hq, d, generator=gen).bfloat16().cuda()
        sn = torch.randint(-1, 6, (S, hkv, 3), generator=gen, dtype=torch.int32).cuda()
        got = nsa.nsa_decode(qn, cache, pages, lens, sn, window=128, cmp_cache=cmp_cache, cmp_pages=cmp_pages, cmp_lens=cmp_lens,
                             gate_w=gate_w)
        qq = qn.double().cpu().numpy()
        c, p, l = (x.cpu().numpy() for x in (cache, pages, lens))
        refs = [oc.attend(qq, cmp_cache.cpu().numpy(), cmp_pages.cpu().numpy(), cmp_lens.cpu().numpy()),
                oc.attend(qq, c, p, l, sn.cpu().numpy()), oc.attend(qq, c, p, l, window=128)]
        want = sum(w * r[0] for w, r in zip(g, refs))
        tol = sum(w * _tolerances(*r, d, torch.float32)[0] for w, r in zip(g, refs)) + 2.0**-22 * np.abs(want)
        assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()
    # the compressed keys that the steps appended are the means of what the cache holds
    Kc, _ = ops.cache_read(cmp_cache, d, cmp_pages, cmp_lens, torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), 2, torch.float32)
    for s in range(S):
        t = (int(cmp_lens[s]) - 1) * 16 + 32
        one = torch.tensor([0, 32], dtype=torch.int32, device="cuda")
        Ks, _ = ops.cache_read(cache, d, pages[s:s + 1].contiguous(), torch.tensor([t], dtype=torch.int32, device="cuda"), one, 32, torch.float32)
        mean = Ks[0].mean(1).bfloat16()
        np.testing.assert_array_equal(Kc[0, :, s].double().cpu().numpy(), oc.values(*oc.quantise(mean.double().cpu().numpy())))


def test_steps_of_several_tokens_lose_no_compressed_key():
    """A prompt in pieces, then drafted tokens that pass the borders of compressed keys between two calls, on caches whose
    empty places are NaN: after each write cache_compress gives every key that it counts, and the decode step is finite."""
    gen = _gen(31)
    hq, hkv, dims, S, W = 8, 2, (64, 64), 3, 6
    cache = torch.full((S * W, hkv, 36 * 128), 0xFF, dtype=torch.uint8, device="cuda")
    cmp_cache = torch.full((4, hkv, 36 * 128), 0xFF, dtype=torch.uint8, device="cuda")
    pages = torch.randperm(S * W, generator=gen).view(S, W).int().cuda()
    cmp_pages = torch.tensor([[3], [0], [2]], dtype=torch.int32, device="cuda")
    lens = torch.zeros(S, dtype=torch.int32, device="cuda")
    for new in ([200, 31, 0], [3, 1, 47], [14, 3, 1], [5, 17, 0], [0, 0, 0], [33, 16, 100]):
        n = sum(new) + 2
        cu = torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device="cuda")
        lens = lens + torch.tensor(new, dtype=torch.int32, device="cuda")
        k, v = (torch.randn(n, hkv, 64, generator=gen).bfloat16().cuda() for _ in range(2))
        ops.cache_write(cache, k, v, pages, lens, cu)
        count = nsa.cache_compress(cache, 64, pages, lens, cmp_cache, cmp_pages, cu_seqlens=cu, n_tokens=n)
        assert count.tolist() == [max(0, (x - 32) // 16 + 1) for x in lens.tolist()]
        whole = torch.tensor([0, *np.cumsum(lens.tolist())], dtype=torch.int32, device="cuda")
        K, V = ops.cache_read(cache, 64, pages, lens, whole, int(whole[-1]), torch.float32)
        cmp_cu = torch.tensor([0, *np.cumsum(count.tolist())], dtype=torch.int32, device="cuda")
        Kc, Vc = ops.cache_read(cmp_cache, 64, cmp_pages, count, cmp_cu, int(cmp_cu[-1]), torch.float32)
        for s in (x for x in range(S) if count[x] > 0):
            at, to = slice(int(whole[s]), int(whole[s + 1])), slice(int(cmp_cu[s]), int(cmp_cu[s + 1]))
            for got, mean in zip((Kc, Vc), nsa.compress_kv(K[:, :, at], V[:, :, at])):
                np.testing.assert_array_equal(got[0, :, to].double().cpu().numpy(),
                                              oc.values(*oc.quantise(mean[0].bfloat16().double().cpu().numpy())))
        sel = torch.zeros(S, hkv, 1, dtype=torch.int32, device="cuda")
        q = torch.randn(S, hq, 64, generator=gen).bfloat16().cuda()
        assert nsa.nsa_decode(q, cache, pages, lens, sel, cmp_cache=cmp_cache, cmp_pages=cmp_pages, cmp_lens=count).isfinite().all()


def _one_group(values, d):
    """Codes and scales of a token whose first group of 16 has `values` in front, all else 0."""
    x = np.zeros((1, d))
    x[0, :len(values)] = values
    return [a[0] for a in oc.quantise(x)]


def _records(tokens, hkv, d_qk, d_v):
    """Pages uint8 [n, hkv, record] of (k values, v values) a token, the same for every head."""
    num = (len(tokens) + 63) // 64
    parts = [np.zeros((num, hkv, 64, w), np.uint8) for w in (d_qk // 2, d_qk // 16, d_v // 2, d_v // 16)]
    for t, (k, v) in enumerate(tokens):
        for i, (x, d) in enumerate(((k, d_qk), (v, d_v))):
            code, byte = _one_group(x, d)
            parts[2 * i][t // 64, :, t % 64] = code[0::2] + 16 * code[1::2]
            parts[2 * i + 1][t // 64, :, t % 64] = byte
    return np.concatenate([p.reshape(num, hkv, -1) for p in parts], -1)


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("n,length,hq,plan", [
    (1000, 640, 1, dict(cluster=1)),                 # a warp for each row
    (3, 640, 4, dict(cluster=2)),
    (100, 1500, 16, dict(cluster=1)),                # teams
    (1, 40000, 9, dict(merge=8)),                    # cut
])
def test_a_long_flat_tail_counts(dims, n, length, hq, plan):
    """One key far above all others, whose values are zeros: O is what the tail adds up to, however small each of its
    weights is.  P is in fp16 at 2^7 times the weight or more (the largest weight is 1), so 2^-25 of it are 2^-32 a key."""
    got_plan = _plan(n, hq, 1, dims, (length + 63) // 64, 0, 64, 0)
    assert {k: got_plan[k] for k in plan} == plan
    num = (length + 63) // 64
    pages3 = torch.from_numpy(_records([([6.0], [0.0])] + [([0.0], [6.0, -1.5, 4.0])] * 127, 1, *dims))
    pages = torch.ones(n, num, dtype=torch.int32)    # (the tail's pages are one page)
    pages[:, 0] = 0
    lens = torch.full((n,), length, dtype=torch.int32)
    q = torch.zeros(n, hq, dims[0])
    q[:, :, 0] = torch.linspace(2, 33, n * hq).view(n, hq) * np.log(2.0) * dims[0]**0.5 / 6   # the tail's weights: 2^-2 to 2^-33
    q = q.bfloat16()
    qd, cd, pd, ld = _cuda(q, pages3, pages, lens)
    out = torch.empty(n, hq, dims[1], device="cuda")
    o, lse = ops.cache_attend(qd, cd, pd, ld, out=out)
    z = q[:, :, 0].double().numpy() * 6 / dims[0]**0.5
    p = np.exp(-z) * (length - 1)
    v = np.zeros(dims[1])
    v[:3] = 6.0, -1.5, 4.0
    want = (p / (1 + p))[..., None] * v
    u = 2.0**-24
    dz = (3 * dims[0] + 8) * u * z                   # (the terms of _tolerances, with 2^-32 for 2^-25)
    rel = 2.0**-11 + 2 * (2.0**-22 + dz) + 4 * length * u + 2.0**-22
    tol = np.abs(want) * (rel[..., None] + u) + length * np.abs(v) * 2.0**-32
    assert (np.abs(o.double().cpu().numpy() - want) <= tol).all()
    ref = z + np.log1p(p)
    assert (np.abs(lse.double().cpu().numpy() - ref) <= dz + 2.0**-22 + dz + 2 * length * u + 2.0**-22 + 8 * u * np.abs(ref)).all()


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq", [3, 16])
@pytest.mark.parametrize("length,width", [(70, 2), (3000, 47), (3000, 1000)])
def test_scores_beyond_a_sums_last_bit(dims, dtype, hq, length, width):
    """Scores so large that half of their last bit is above fp16's range in powers of two: the key far above the others has
    all of the weight, in its page and behind it, and two equal ones in one page have half of it each."""
    gen = _gen(60)
    top, twin, d = length // 2 // 64 * 64 + 5, length // 2 // 64 * 64 + 9, dims[0]
    size = torch.exp2(torch.arange(hq).float() * 5 / hq + 10) * (1 + torch.rand(hq, generator=gen))   # scores of 2^28 to 2^35
    q = size.view(hq, 1).expand(2, hq, d).to(dtype)
    k, v = torch.zeros(2 * length, 1, d), torch.randn(2 * length, 1, dims[1], generator=gen)
    for s in range(2):
        k[s * length:(s + 1) * length, 0] = torch.rand(length, 1, generator=gen) * 20000
        k[s * length + top] = 60000.0
    k[length + twin] = 60000.0
    pages, lens, cu = _batch([length] * 2, [length] * 2, 2 * ((length + 63) // 64), gen, width)
    cache = ops.cache_alloc(2 * ((length + 63) // 64), 1, *dims)
    kd, vd, pd, ld, cd, qd = _cuda(k.to(dtype), v.to(dtype), pages, lens, cu, q)
    ops.cache_write(cache, kd, vd, pd, ld, cd)
    K, V = (x[0, 0].double().cpu().numpy() for x in ops.cache_read(cache, d, pd, ld, cd, 2 * length, torch.float32))
    assert (np.sort(K[:length, 0])[-2] < 0.5 * K[top, 0]) and K[length + top, 0] == K[length + twin, 0]
    want = np.stack((V[top], (V[length + top] + V[length + twin]) / 2))
    ref = q[:, :, 0].double().numpy() * K[top, 0] * d**0.5 + np.log([[1.0], [2.0]])
    o, lse = ops.cache_attend(qd, cache, pd, ld, out=torch.empty(2, hq, dims[1], device="cuda"))
    got = o.double().cpu().numpy()
    # (every P is 0 or one power of two: 2^-22 for that in the sum, 2^-22 for the division and weight)
    assert (np.abs(got - want[:, None]) <= np.abs(V).max() * 2.0**-21).all()
    assert (np.abs(lse.double().cpu().numpy() - ref) <= (3 * d + 8) * 2.0**-24 * np.abs(ref)).all()


@pytest.mark.parametrize("case", [0, 4, 6, 7, 10, 12, 13, 14])
def test_waits_are_bounded_however_the_work_is_shared(case):
    """No copy comes: the launch ends by itself, every row that has a key is NaN through each kind of join, the error word is
    set, and the next call is right."""
    lens, width, n_sel, dims, (hq, hkv), want_plan = SHARING[case]
    n = len(lens)
    gen = _gen(70 + case)
    num_pages = sum((x + 63) // 64 for x in lens)
    pages, lens, _ = _batch(lens, None, num_pages, gen, width)
    cache = _random_cache(num_pages, hkv, dims, gen)
    q = torch.randn(n, hq, dims[0], generator=gen).bfloat16()
    sel = torch.randint(-1, width, (n, hkv, n_sel), generator=gen, dtype=torch.int32) if n_sel else None
    if n_sel:
        sel[:, :, 0] = torch.clamp(lens - 1, min=0).view(-1, 1) // 64
    qd, cd, pd, ld, sd = _cuda(q, cache, pages, lens, sel)
    want = ops.cache_attend(qd, cd, pd, ld, sel=sd)
    o, lse, err = torch.zeros_like(want[0]), torch.zeros_like(want[1]), torch.zeros(1, dtype=torch.int32, device="cuda")
    batch = capi.make_cache_batch(cache=cd.data_ptr(), pages=pd.data_ptr(), lens=ld.data_ptr(), num_pages=num_pages, n_seqs=n,
                                  width=width, n_rows=n, heads_kv=hkv, d_qk=dims[0], d_v=dims[1])
    desc = capi.make_cache_attend_desc(batch=batch, q=qd.data_ptr(), o=o.data_ptr(), lse=lse.data_ptr(), heads_q=hq,
                                       sel=sd.data_ptr() if n_sel else 0, n_sel=n_sel, block_size=64, err=err.data_ptr(),
                                       timeout_ms=20, debug_flags=capi.NSA_DEBUG_STALL)
    plan = capi.cache_attend_plan(desc, 0)
    assert {k: plan[k] for k in want_plan} == want_plan
    work = torch.empty(capi.cache_attend_workspace_bytes(desc), dtype=torch.uint8, device="cuda")
    desc.workspace = work.data_ptr()
    stream = torch.cuda.current_stream().cuda_stream
    capi.cache_attend(desc, stream)
    assert err.item() == capi.NSA_DEVERR_TIMEOUT
    live = ld > 0
    assert o[live].isnan().all() and lse[live].isnan().all()
    assert not o[~live].any() and torch.isneginf(lse[~live]).all()
    err.zero_()
    desc.debug_flags = 0
    capi.cache_attend(desc, stream)
    assert err.item() == 0 and torch.equal(o, want[0]) and torch.equal(lse, want[1])


def test_a_wait_that_ran_out_is_told_through_torch():
    q, cache, pages, lens = _small(27)
    err = torch.tensor([4, 9], dtype=torch.int32, device="cuda")
    want = ops.cache_attend(q, cache, pages, lens, err=err)
    assert err.tolist() == [4, 9]
    sel = torch.zeros(3, 2, 1, dtype=torch.int32, device="cuda")
    nsa.nsa_decode(q, cache, pages, lens, sel, err=err)
    assert err.tolist() == [4, 9]
    o, _ = ops._C.cache_attend(q, cache, pages, lens, err=err, timeout_ms=20, debug_flags=capi.NSA_DEBUG_STALL)
    assert o.isnan().all() and err.tolist() == [4 | capi.NSA_DEVERR_TIMEOUT, 9]
    assert torch.equal(ops.cache_attend(q, cache, pages, lens)[0], want[0])
    for bad in (err.long(), err.cpu(), err[:0]):
        with pytest.raises(RuntimeError, match="err must be"):
            ops.cache_attend(q, cache, pages, lens, err=bad)


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_value_of_the_type_is_quantised_by_the_definition(dtype):
    """Every finite value as the largest of a group, and for each scale every value that is not beyond its saturation and not
    far below its first border, with either sign: the kernel's bytes are the oracle's."""
    every = torch.arange(0x7F80 if dtype == torch.bfloat16 else 0x7C00, dtype=torch.int16).view(dtype)
    groups = torch.zeros(len(every), 16, dtype=dtype)
    groups[torch.arange(len(every)), torch.arange(len(every)) % 16] = every * (1 - 2 * (torch.arange(len(every)) // 16 % 2)).to(dtype)
    parts, x = [groups], every.double().numpy()
    taken = oc.quantise(np.concatenate((x[:, None], np.zeros((len(x), 15))), 1))[1][:, 0]   # the scale of each as the largest
    for byte in range(1, 0xE3):
        if not (taken == byte).any():
            continue
        lead = every[np.nonzero(taken == byte)[0].max() if byte < 0xE2 else int(np.searchsorted(x, 6 * 10240.0))]
        below = every[torch.from_numpy((x >= 0.2 * oc._SCALES[byte]) & (x <= float(lead)))]
        below = torch.cat((below, below.new_zeros(-len(below) % 15))).view(-1, 15)
        parts.append(torch.cat((lead.expand(len(below), 1), below), 1))
        parts.append(-parts[-1].flip(1))
    x = torch.cat(parts)
    x = torch.cat((x, x.new_zeros(-len(x) % 8, 16))).view(-1, 1, 128)
    n = x.shape[0]
    cache = ops.cache_alloc((n + 63) // 64, 1, 128, 128)
    pages = torch.arange(cache.shape[0], dtype=torch.int32, device="cuda")[None]
    lens, cu = torch.tensor([n], dtype=torch.int32, device="cuda"), torch.tensor([0, n], dtype=torch.int32, device="cuda")
    ops.cache_write(cache, x.cuda(), x.flip(0).contiguous().cuda(), pages, lens, cu)
    code, byte = oc.quantise(x[:, 0].double().numpy())
    kc, ks, vc, vs = (p[:, 0].reshape(-1, p.shape[-1])[:n] for p in oc.split(cache.cpu().numpy(), 128, 128))
    for codes, scales, c, b in ((kc, ks, code, byte), (vc, vs, code[::-1], byte[::-1])):
        np.testing.assert_array_equal(scales, b)
        got = np.stack((codes & 15, codes >> 4), -1).reshape(n, 128)
        assert ((got == c) | ((got & 7 == 0) & (c & 7 == 0))).all()          # (the sign of a zero is free)


def test_a_captured_step_of_several_tokens_compresses_on_replay(monkeypatch):
    """Write and compress captured once, replayed on other lengths, rows and keys, each a chunk of three compressed keys at a
    time: the same caches as by calls that are not captured and take all at once."""
    gen = _gen(32)
    hkv, S, W, n = 2, 3, 8, 70
    pages = torch.randperm(S * W, generator=gen).view(S, W).int().cuda()
    cmp_pages = torch.tensor([[1], [2], [0]], dtype=torch.int32, device="cuda")
    size = lambda p: torch.full((p, hkv, 36 * 192), 0xFF, dtype=torch.uint8, device="cuda")  # noqa: E731
    caches, want = (size(S * W), size(3)), (size(S * W), size(3))
    lens, cu = torch.zeros(S, dtype=torch.int32, device="cuda"), torch.zeros(S + 1, dtype=torch.int32, device="cuda")
    k, v = torch.zeros(n, hkv, 128, device="cuda").half(), torch.zeros(n, hkv, 64, device="cuda").half()

    def step(cache, cmp_cache):
        ops.cache_write(cache, k, v, pages, lens, cu)
        return nsa.cache_compress(cache, 128, pages, lens, cmp_cache, cmp_pages, cu_seqlens=cu, n_tokens=n)

    monkeypatch.setattr(nsa, "COMPRESS_VALUES", 3 * 32 * hkv * 192)
    step(*caches)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        count = step(*caches)
    monkeypatch.undo()
    for new in ([60, 0, 10], [1, 2, 3], [0, 0, 70], [16, 32, 8], [0, 0, 0], [15, 17, 33]):
        cu.copy_(torch.tensor([0, *np.cumsum(new)], dtype=torch.int32))
        lens += torch.tensor(new, dtype=torch.int32, device="cuda")
        k.copy_(torch.randn(n, hkv, 128, generator=gen))
        v.copy_(torch.randn(n, hkv, 64, generator=gen))
        g.replay()
        assert torch.equal(count, step(*want))
        torch.cuda.synchronize()
        assert torch.equal(caches[0], want[0]) and torch.equal(caches[1], want[1])
    assert count.tolist() == [max(0, (x - 32) // 16 + 1) for x in lens.tolist()]
    back, _ = ops.cache_read(caches[1], 128, cmp_pages, count, torch.tensor([0, *np.cumsum(count.tolist())], dtype=torch.int32,
                                                                           device="cuda"), int(count.sum()))
    assert back.isfinite().all()
