"""Edges of a decode step's preparation on the GPU: block selection from queries whose channels are far apart and
from the longest sequences, against the oracle's exact sums;
forward-mode derivatives of the rotary positions, and where their gradients lie; pages of the compressed cache."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from nsa_hopper_b200 import capi, nsa, ops
from oracle import cache as oc
from oracle import step as oracle
from tests.test_gpu_step import DIMS, _check_select, _records, _t, _tables

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ block selection
@pytest.mark.parametrize("dims,hq,hkv,n_sel,top", [(DIMS[1], 16, 1, 16, 36), (DIMS[1], 16, 1, 16, 44), (DIMS[0], 1, 1, 40, 44),
                                                   (DIMS[2], 10, 2, 300, 60), (DIMS[0], 256, 1, 7, 100)])
def test_select_of_a_query_with_a_far_channel(dims, hq, hkv, n_sel, top):
    """One channel of 2^top, whose keys are zero, and channels of 1 that decide: its products are 0 exactly, those of the others and
    their sums in fp64 lose 2^-50 of the scores, which are 2^-10 apart and more but for one pair in 10^10."""
    g = torch.Generator().manual_seed(top + hq)
    lens = [65536 if hkv == 1 else 30000, 700, 40]
    pages, count = _tables(lens, 32, 16, np.random.default_rng(top))
    x = torch.randn(count, hkv, 64, dims[0], generator=g)
    x[..., 5] = 0
    q = torch.randn(len(lens), hq, dims[0], generator=g)
    q[:, hq // 2, 5] = 2.0**top
    q[1, 0, 5] = -2.0**top
    _check_select(q.to(torch.bfloat16), _records(x, dims[1]), pages, lens, n_sel)


@pytest.mark.parametrize("dims", DIMS[:3])
def test_select_of_many_rows_with_far_channels(dims):
    """The same where blocks of the second kernel are small; every second row's channels are alike."""
    rng, g = np.random.default_rng(dims[0]), torch.Generator().manual_seed(dims[0])
    lens = rng.integers(1, 1500, 200)
    pages, count = _tables([1500], 32, 16, rng)
    pages = np.stack([np.roll(pages[0], r) for r in range(len(lens))])
    x = torch.randn(count, 4, 64, dims[0], generator=g)
    x[..., 40] = 0
    q = torch.randn(len(lens), 8, dims[0], generator=g)
    q[::2, 1::2, 40] = -2.0**50
    q[::4, 1, 40] = 2.0**-100  # (far below: lost by none of the sums, as its keys are zero)
    _check_select(q.to(torch.bfloat16), _records(x, dims[1]), pages, lens, 9)


def test_select_of_fp16_numbers_from_the_smallest_to_the_largest():
    """256 heads leave the whole numbers 38 bits, of which fp16 has 40."""
    g = torch.Generator().manual_seed(3)
    lens = [5000, 64]
    pages, count = _tables(lens, 32, 16, np.random.default_rng(4))
    x = torch.randn(count, 1, 64, 64, generator=g)
    x[..., 63] = 0
    q = torch.randint(-3, 4, (2, 256, 64), generator=g) * 2.0**-24
    q[:, 17, 63] = 65504.0
    _check_select(q.to(torch.float16), _records(x, 64), pages, lens, 12)


def test_select_of_many_launches_in_the_workspace_of_one():
    """2300 rows with the workspace that is asked for and not a byte more, against calls of few rows."""
    g = torch.Generator().manual_seed(14)
    rows, count = 2300, 5
    lens = np.random.default_rng(14).integers(0, 900, rows)
    pages = _t(np.random.default_rng(15).integers(0, count, (rows, 1)))
    cache = torch.from_numpy(_records(torch.randn(count, 2, 64, 64, generator=g), 64)).cuda()
    q, lens = torch.randn(rows, 4, 64, generator=g).to("cuda", torch.bfloat16), _t(lens)
    batch = capi.make_cache_batch(cache=cache.data_ptr(), pages=pages.data_ptr(), lens=lens.data_ptr(), num_pages=count, n_seqs=rows,
                                  width=1, n_rows=rows, heads_kv=2, d_qk=64, d_v=64)
    sel = torch.full((rows, 2, 6), 7, dtype=torch.int32, device="cuda")
    desc = capi.make_cache_select_desc(batch=batch, q=q.data_ptr(), sel=sel.data_ptr(), heads_q=4, n_sel=6, block_size=64, cmp_block=32,
                                       cmp_stride=16, q_dtype=capi.DTYPE_BF16)
    size = capi.cache_select_workspace_bytes(desc)
    assert size == 1024 * 2 * 17 * 8  # (T up to 64 * 16 + 31 = 1055 tokens, 17 blocks)
    work = torch.full((size + 4096,), 0xAB, dtype=torch.uint8, device="cuda")
    desc.workspace = work.data_ptr()
    capi.cache_select(desc, torch.cuda.current_stream().cuda_stream)
    want = torch.cat([ops.cache_select(q[r:r + 500], cache, pages[r:r + 500], lens[r:r + 500], 6) for r in range(0, rows, 500)])
    assert torch.equal(sel, want) and (work[size:] == 0xAB).all()


def test_select_of_several_passes():
    """300000 tokens: 4688 blocks in three passes of 2048, 293 pages of keys, more than are looked up beforehand.  Pages of equal
    keys stand at the first pass's end and the next one's beginning, in the middle and at the end, so that equal scores meet
    across passes; a row of other keys throughout; lengths that end with a pass and behind it."""
    rng, g = np.random.default_rng(16), torch.Generator().manual_seed(16)
    lens = [300000, 300000, 131072, 131073, 262144 + 31]
    pages, _ = _tables(lens, 32, 16, rng)
    assert pages.shape[1] == 293
    x = torch.randn(24, 1, 64, 64, generator=g)
    x[:4] = x[:4, :, :1]  # (pages of one key 64 times)
    q = torch.randn(5, 4, 64, generator=g).to(torch.bfloat16)
    x[2] = (q[0].float().sum(0) / 8).expand(64, 64)  # (what row 0 looks for)
    for r in (0, 2, 3, 4):
        pages[r] = np.where(pages[r] >= 0, rng.integers(0, 2, pages.shape[1]), -1)
    pages[0, [3, 127, 128, 150, 200, 255, 256, 257, 291, 292]] = 2
    pages[1] = rng.integers(4, 24, pages.shape[1])
    cache = _records(x, 64)
    want = oracle.select(q.double().numpy(), cache, pages, np.array(lens), 1024)
    passes = {int(b) // 2048 for b in want[0, 0, :100]}
    assert passes == {0, 1, 2} and {int(b) // 2048 for b in want[1, 0]} == passes and (want >= 0).all()
    args = q.cuda(), torch.from_numpy(cache).cuda(), _t(pages), _t(lens)
    for n_sel in (1, 16, 100, 1024):
        assert np.array_equal(ops.cache_select(*args, n_sel).cpu().numpy(), want[..., :n_sel])


def test_select_of_the_longest_sequences():
    """2^24 tokens, the most that float32 places: a million keys, mostly zeros, of whole numbers; one token more selects nothing."""
    rng, g = np.random.default_rng(17), torch.Generator().manual_seed(17)
    most, width, n_sel = 2**24, 16384, 40
    lens = [most, most + 1, most - 5, 31]
    x = torch.zeros(6, 1, 64, 64)
    x[1:] = torch.randint(-6, 7, (5, 1, 64, 64), generator=g).clamp(-4, 4)
    x[1:, ..., ::16] = 6  # (so that every scale is 1)
    cache = _records(x, 64)
    keys, _ = oc.decode(cache[:, 0], 64, 64)
    assert np.array_equal(keys, x[:, 0].numpy())
    pages = np.where(rng.random((4, width)) < 0.01, rng.integers(1, 6, (4, width)), 0).astype(np.int32)
    pages[:, [0, 127, 128, 8191, 16383]] = 5
    q = torch.randint(-9, 10, (4, 3, 64), generator=g).to(torch.bfloat16)
    got = ops.cache_select(q.cuda(), torch.from_numpy(cache).cuda(), _t(pages), _t(lens), n_sel).cpu().numpy()
    for r, tokens in enumerate(lens):
        if tokens > most:
            assert (got[r] == -1).all()
            continue
        n, blocks = oracle.completed(tokens, 32, 16), -(-tokens // 64)
        score = np.zeros(blocks)
        if n:
            where = np.floor(torch.linspace(0, tokens - 1, n, dtype=torch.float32).numpy() / 64).astype(np.int64)
            np.add.at(score, np.minimum(where, blocks - 1), (keys @ q[r].double().sum(0).numpy())[pages[r]].ravel()[:n])
        want = np.argsort(-score, kind="stable")[:n_sel]
        assert got[r, 0].tolist() == want.tolist() + [-1] * (n_sel - len(want))
        assert r == 1 or n == 0 or {int(b) // 2048 for b in want} > {int(want[0]) // 2048}


# ------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize("layout", ["rows", "tokens"])
@pytest.mark.parametrize("leaves", [False, True])
def test_rotary_in_forward_mode(layout, leaves):
    """The turn is linear: an output's tangent is the turned tangent, bit for bit what a call with it gives."""
    g = torch.Generator().manual_seed(6)
    plan = ops.rotary_plan(24, rotary_dim=16, offset=4)
    shape = (6, 3, 24) if layout == "rows" else (2, 6, 3, 24)
    pos = torch.randint(0, 5000, shape[:-2], generator=g).int().cuda()
    view = (lambda t: t.transpose(1, 2)) if layout == "tokens" else (lambda t: t)
    x, dx, y, dy = (view(torch.randn(shape, generator=g).cuda()) for _ in range(4))
    want, moved = ops.rotary(x, y, pos, plan), ops.rotary(dx, dy, pos, plan)
    if leaves:
        x, y = x.requires_grad_(), y.requires_grad_()
    with forward_ad.dual_level():
        a, b = forward_ad.make_dual(x, dx), forward_ad.make_dual(y, dy)

        def same(got, value, tangent):
            u = forward_ad.unpack_dual(got)
            assert torch.equal(u.primal, value) and (u.tangent is None) == (tangent is None)
            assert tangent is None or torch.equal(u.tangent, tangent)
            assert got.requires_grad == leaves

        for q, k in ((a, b), (a, y), (x, b)):
            u, v = ops.rotary(q, k, pos, plan)
            same(u, want[0], moved[0] if q is a else None)
            same(v, want[1], moved[1] if k is b else None)
        alone, none = ops.rotary(a, None, pos, plan)
        assert none is None
        same(alone, want[0], moved[0])
        if leaves:  # reverse over forward: the gradient of what the tangent does not depend on, and of the primal
            (grad,) = torch.autograd.grad(forward_ad.unpack_dual(alone).primal, x, dx)
            assert torch.equal(grad, ops.rotary(dx, None, pos, plan, inverse=True)[0])
    assert forward_ad.unpack_dual(ops.rotary(x, y, pos, plan)[0]).tangent is None


def test_rotary_gradients_in_forward_mode():
    """Forward over reverse: the tangent of a gradient is the turn back of the incoming gradient's tangent."""
    g = torch.Generator().manual_seed(7)
    plan, pos = ops.rotary_plan(16), torch.arange(5, dtype=torch.int32, device="cuda")
    x = torch.randn(5, 2, 16, generator=g).cuda().requires_grad_()
    d, t = (torch.randn(5, 2, 16, generator=g).cuda() for _ in range(2))
    y, _ = ops.rotary(x, None, pos, plan)
    with forward_ad.dual_level():
        (grad,) = torch.autograd.grad(y, x, forward_ad.make_dual(d, t))
        u = forward_ad.unpack_dual(grad)
        assert torch.equal(u.primal, ops.rotary(d, None, pos, plan, inverse=True)[0])
        assert torch.equal(u.tangent, ops.rotary(t, None, pos, plan, inverse=True)[0])


@pytest.mark.parametrize("parts", [(4, 2, 2), (1, 1, 1), (3, 0, 5)])
def test_rotary_gradients_lie_as_a_fused_projection(parts):
    """Heads cut out of a fused projection: gradients have its order of tokens and heads, and the values of whole tensors."""
    g = torch.Generator().manual_seed(sum(parts))
    B, T, d, (hq, hk, _) = 2, 6, 16, parts
    plan, pos = ops.rotary_plan(d), torch.arange(T, dtype=torch.int32, device="cuda").expand(B, T)
    fused = torch.randn(B, T, sum(parts), d, generator=g).cuda().requires_grad_()
    q, k = fused[:, :, :hq].transpose(1, 2), fused[:, :, hq:hq + hk].transpose(1, 2) if hk else None
    out = [x for x in ops.rotary(q, k, pos, plan) if x is not None]
    grads = [torch.randn(x.shape, generator=g).cuda() for x in out]
    views = [x for x in (q, k) if x is not None]
    back = torch.autograd.grad(out, views, grads, retain_graph=True)
    for x, y, dy in zip(views, back, grads):
        assert y.transpose(1, 2).is_contiguous() and torch.equal(y, ops.rotary(dy, None, pos, plan, inverse=True)[0])
    (whole,) = torch.autograd.grad(out, fused, grads)
    assert torch.equal(whole[:, :, :hq], back[0].transpose(1, 2)) and (whole[:, :, hq + hk:] == 0).all()
    x = q.detach().contiguous().requires_grad_()  # (heads one after the other)
    (y,) = torch.autograd.grad(ops.rotary(x, None, pos, plan)[0], x, grads[0])
    assert y.is_contiguous() and torch.equal(y, back[0])


# ------------------------------------------------------------------ whole steps
@pytest.mark.parametrize("captured", [False, True])
def test_steps_whose_compressed_pages_come_from_a_pool(captured):
    """The second pool runs out: the sequence that completes a key has no rows until another one has ended, no page is in two
    rows of a table, and outputs are those of a fixed table for the compressed keys.  Rejected drafts are given back in a
    call of their own."""
    g = torch.Generator().manual_seed(31)
    S, hq, hk, d, width, wide, n_sel = 4, 4, 2, 64, 36, 3, 3
    i32 = dict(dtype=torch.int32, device="cuda")
    prompt = [1055, 500, 2075, 31]  # 64, 30, 128 and 0 compressed keys: 4 pages
    plan, total, cmp_count = ops.rotary_plan(d), sum(prompt), 5
    pages, held, pool, n_free = torch.full((S, width), -1, **i32), torch.zeros(S, **i32), torch.randperm(S * width, generator=g).int().cuda(), _t([S * width])
    cmp_pages, cmp_held, cmp_pool, cmp_free = (torch.full((S, wide), -1, **i32), torch.zeros(S, **i32),
                                               torch.randperm(cmp_count, generator=g).int().cuda(), _t([cmp_count]))
    fixed = torch.arange(S * wide, **i32).view(S, wide)
    cache, cmp_cache, cmp_fixed = ops.cache_alloc(S * width, hk, d, d), ops.cache_alloc(cmp_count, hk, d, d), ops.cache_alloc(S * wide, hk, d, d)
    rows = _t(prompt)

    def reserve(n_tokens=None):
        batch = ops.cache_reserve(pages, held, rows, pool, n_free, n_tokens=n_tokens)
        want = torch.where(held >= 32, (held - 32) // 16 + 1, 0)
        ops.cache_reserve(cmp_pages, cmp_held, want - cmp_held, cmp_pool, cmp_free)
        short = cmp_held != want
        ops.cache_reserve(pages, held, torch.where(short, -rows, 0), pool, n_free)
        return batch._replace(lens=torch.where(short, 0, batch.lens))

    batch = reserve(total)
    assert batch.lens.tolist() == prompt == held.tolist() and cmp_held.tolist() == [64, 30, 128, 0] and int(cmp_free) == 1
    k, v = (torch.randn(total, hk, d, generator=g).to("cuda", torch.bfloat16) for _ in range(2))
    _, k = ops.rotary(k[:, :1], k, batch.positions, plan)
    ops.cache_write(cache, k, v, pages, batch.lens, cu_seqlens=batch.cu_seqlens)
    for c, p in ((cmp_cache, cmp_pages), (cmp_fixed, fixed)):
        nsa.cache_compress(cache, d, pages, batch.lens, c, p, cu_seqlens=batch.cu_seqlens, n_tokens=total)
    q, k, v = (torch.randn(S, h, d, generator=g).to("cuda", torch.bfloat16) for h in (hq, hk, hk))

    def step():
        batch = reserve()
        a, b = ops.rotary(q, k, batch.positions, plan)
        ops.cache_write(cache, b, v, pages, batch.lens)
        out = []
        for c, p in ((cmp_cache, cmp_pages), (cmp_fixed, fixed)):
            cmp_lens = nsa.cache_compress(cache, d, pages, batch.lens, c, p)
            out.append(nsa.nsa_decode(a, cache, pages, batch.lens, window=64, cmp_cache=c, cmp_pages=p, cmp_lens=cmp_lens, n_sel=n_sel))
            out.append(ops.cache_select(a, c, p, batch.lens, n_sel))
        return batch, out

    graph, results = torch.cuda.CUDAGraph(), None
    if captured:
        state = [pages, held, pool, n_free, cmp_pages, cmp_held, cmp_pool, cmp_free, cache, cmp_cache, cmp_fixed]
        saved = [t.clone() for t in state]
        rows.copy_(_t([1, 1, 1, 0]))
        step()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            results = step()
        for t, old in zip(state, saved):
            t.copy_(old)
    have = list(prompt)
    # rows of each step, and the sequences whose rows are refused: sequence 0's key 64 and sequence 3's key 0 want the last page
    for asked, refused in (([0, 1, 1, 1], []), ([1, 1, 1, 1], [0]), ([1, 0, 0, 1], [0]), ([0, -502, 1, 0], []), ([1, 0, 1, 1], []),
                           ([0, 0, -1030, 0], []), ([1, 1, 1, 0], [])):
        rows.copy_(_t(asked))
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        if captured:
            graph.replay()
        batch, (out, sel, want, want_sel) = results if captured else step()
        have = [max(0, n + r) if s not in refused else n for s, (n, r) in enumerate(zip(have, asked))]
        assert held.tolist() == have and cmp_held.tolist() == [oracle.completed(n, 32, 16) for n in have]
        assert batch.lens.tolist() == [n if r > 0 and s not in refused else 0 for s, (n, r) in enumerate(zip(have, asked))]
        for table, h, p, n in ((pages, held, pool, n_free), (cmp_pages, cmp_held, cmp_pool, cmp_free)):
            ids = [i for s in range(S) for i in table[s, :-(-int(h[s]) // 64)].tolist()] + p[:int(n)].tolist()
            assert sorted(ids) == list(range(len(p)))
        # (the same keys at other places, and the same shares of the work: equal, but for what fp32 sums may differ by)
        assert torch.equal(sel, want_sel) and float((out - want).abs().max()) <= 2.0**-10 * float(want.abs().max())
        assert ((out != 0).flatten(1).any(1) == (batch.lens > 0)).all()
