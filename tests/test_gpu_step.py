"""Pages, rotary positions and block selection of a decode step on the GPU against the oracle, by themselves and in a run of
whole steps.  Whole numbers are compared for equality."""
import math

import numpy as np
import pytest
import torch

from nsa_hopper_b200 import capi, nsa, ops
from oracle import cache as oc
from oracle import step as oracle
from tests.test_step import random_batch

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")


def _t(x, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x), dtype=dtype, device="cuda")


# ------------------------------------------------------------------ pages
def _check_reserve(pages, held, rows, pool, n_free, n_rows, update, stride=None):
    table = _t(pages)
    if stride:
        wide = torch.full((pages.shape[0], stride), 77, **I32)
        wide[:, :pages.shape[1]] = table
        table = wide[:, :pages.shape[1]]
    state = [table, _t(held), _t(rows), _t(pool), _t([n_free])]
    got = ops.cache_reserve(*state, n_tokens=n_rows, update=update)
    want = oracle.reserve(pages, held, rows, pool, n_free, n_rows)
    assert (got.cu_seqlens is None) == (n_rows is None)
    for name, g, w in zip(("pages", "pool", "lens", "cu", "positions", "slots", "held", "n_free"),
                          (state[0], state[3], got.lens, got.cu_seqlens, got.positions, got.slots, got.held, got.n_free), want):
        assert (w is None and g is None) or np.array_equal(g.cpu().numpy().ravel(), np.asarray(w).ravel()), name
    assert (got.held is state[1]) == update or got.held.data_ptr() == state[1].data_ptr()
    if update:
        assert torch.equal(got.held, state[1]) and torch.equal(got.n_free, state[4])
    else:
        assert np.array_equal(state[1].cpu(), held) and int(state[4]) == n_free
    if stride:
        assert (wide[:, pages.shape[1]:] == 77).all()
    return got


@pytest.mark.parametrize("n,width", [(1, 1), (1, 300), (7, 5), (33, 9), (64, 40), (65, 40), (257, 33), (1000, 7), (1025, 20), (3001, 12)])
@pytest.mark.parametrize("packed", [False, True])
def test_reserve(n, width, packed):
    rng = np.random.default_rng(n + width)
    for update in (False, True):
        pages, held, rows, pool, n_free = random_batch(rng, n, width)
        total = int(np.maximum(rows, 0).sum())
        _check_reserve(pages, held, rows, pool, n_free, total + (5 if update else 0) if packed else None, update,
                       width + 3 if update else None)


@pytest.mark.parametrize("seed", range(6))
def test_reserve_takes_broken_tables(seed):
    rng = np.random.default_rng(seed)
    for case in range(4):
        n, width = int(rng.choice([1, 5, 40, 700])), int(rng.choice([0, 1, 4, 30]))
        pages, held, rows, pool, n_free = random_batch(rng, n, width, broken=True)
        _check_reserve(pages, held, rows, pool, n_free, (None, 3000, 0, 17)[case], bool(seed % 2))


def test_reserve_many_packed_rows():
    """Prompts whose rows take a kernel of their own, the last of them without pages, rows cut off and rows of none."""
    rng = np.random.default_rng(1)
    n, width = 40, 64
    held, rows = rng.integers(0, 70, n).astype(np.int32), rng.integers(1, 2000, n).astype(np.int32)
    rows[7], rows[9], held[11], rows[11] = 0, 5000, 500, -500
    used = -(-held // 64)
    want = int((-(-(held + rows) // 64) - used)[rows > 0].sum())
    pool = rng.permutation(want + int(used.sum())).astype(np.int32)
    pages = np.full((n, width), -1, np.int32)
    at = want - 60
    for s in range(n):
        pages[s, :used[s]] = pool[at:at + used[s]]
        at += used[s]
    total = int(np.maximum(rows, 0).sum())
    assert total > 20000
    for n_rows in (total, total - 777, total + 333):
        got = _check_reserve(pages, held, rows, pool, want - 60, n_rows, False)
        assert int(got.lens[9]) == 0 and (got.positions[:20000] == -1).any()  # (more than a row of the table holds)
        got = _check_reserve(pages, held, rows, pool, want - 300, n_rows, False)  # (and too few pages for the last ones)
        assert (got.lens.cpu().numpy()[rows > 0] == 0).sum() > 1


def test_reserve_largest_batches_and_refusals():
    n = 8192
    pages, held, rows = torch.full((n, 2), -1, **I32), torch.zeros(n, **I32), torch.ones(n, **I32)
    pool, n_free = torch.randperm(n, device="cuda").int(), _t([n])
    order = pool.clone()
    got = ops.cache_reserve(pages, held, rows, pool, n_free)
    assert int(n_free) == 0 and (got.positions == 0).all() and torch.equal(pages[:, 0], order) and (held == 1).all()
    assert torch.equal(got.slots, order.long() * 64) and got.cu_seqlens is None
    got = ops.cache_reserve(pages, held, -held, pool, n_free)
    assert int(n_free) == n and torch.equal(pool, order) and (held == 0).all() and (got.lens == 0).all() and (got.slots == -1).all()
    empty = ops.cache_reserve(pages[:0], held[:0], rows[:0], pool, n_free, n_tokens=3)
    assert empty.lens.shape == (0,) and empty.cu_seqlens.tolist() == [0] and empty.positions.tolist() == [-1] * 3 and int(empty.n_free) == n
    z = torch.zeros(n + 1, **I32)
    with pytest.raises(RuntimeError, match="8192"):
        ops.cache_reserve(torch.zeros(n + 1, 1, **I32), z, z, pool, n_free)
    for bad in (dict(held=held[:5]), dict(rows=rows.long()), dict(pool=pool.view(2, -1)), dict(n_free=pool[:2]), dict(held=held[::2]),
                dict(pages=pages.long()), dict(pages=pages.T), dict(n_tokens=-1), dict(rows=rows.cpu())):
        args = dict(pages=pages, held=held, rows=rows, pool=pool, n_free=n_free)
        with pytest.raises(RuntimeError):
            ops.cache_reserve(**{**args, **bad})


def test_reserve_in_a_graph_with_other_rows():
    """A captured step that replays from what the last one left: state in place, rows written between replays."""
    rng = np.random.default_rng(9)
    n, width, count = 50, 8, 200
    pages, held = np.full((n, width), -1, np.int32), np.zeros(n, np.int32)
    pool, n_free = rng.permutation(count).astype(np.int32), count
    d_pages, d_held, d_rows, d_pool, d_free = _t(pages), _t(held), torch.zeros(n, **I32), _t(pool), _t([n_free])
    ops.cache_reserve(d_pages, d_held, d_rows, d_pool, d_free, n_tokens=6000)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.cache_reserve(d_pages, d_held, d_rows, d_pool, d_free, n_tokens=6000)
    for _ in range(12):
        rows = np.where(rng.random(n) < 0.3, -rng.integers(0, 500, n), rng.integers(0, 120, n)).astype(np.int32)
        d_rows.copy_(_t(rows))
        graph.replay()
        pages, pool, lens, cu, pos, slots, held, n_free = oracle.reserve(pages, held, rows, pool, n_free, 6000)
        held = held.astype(np.int32)
        for g, w in ((d_pages, pages), (d_pool, pool), (got.lens, lens), (got.cu_seqlens, cu), (got.positions, pos), (got.slots, slots),
                     (d_held, held)):
            assert np.array_equal(g.cpu().numpy(), w)
        assert int(d_free) == n_free


# ------------------------------------------------------------------ rotary positions
def _tolerance(size, want, dtype):
    """cos and sin: the angle is off by 2^-32 of a turn and half a step of fp32 of at most pi / 4, sincospi by two steps:
    less than 4 half steps of 1.  Two products and a sum: two half steps more of |a| + |b|.  Then half a step of the type."""
    return 6 * 2.0**-24 * size + torch.finfo(dtype).eps / 2 * np.abs(want) + (2.0**-25 if dtype == torch.float16 else 0.0)


def _freqs(dim, base=1e4):
    return oracle.plan_frequencies(dim, base)


def _check_rotary(x, got, pos, plan, freqs, inverse=False):
    """x, got [..., H, d] (any device layout), pos numpy [axes, ...]."""
    angle = oracle.angles(pos, freqs, plan.axis.tolist())
    want, size = oracle.rotary(x.detach().double().cpu().numpy(), angle, plan.offset, plan.interleaved, inverse)
    err = np.abs(got.detach().double().cpu().numpy() - want)
    tol = _tolerance(size, want, got.dtype)
    assert (err <= tol).all(), (np.argwhere(err > tol)[:3], err.max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,dim,offset,sections", [(128, 128, 0, (16, 24, 24)), (192, 64, 128, (32,)), (72, 72, 0, (18, 18)), (64, 36, 28, (5, 6, 7)),
                                                   (256, 256, 0, (1, 126, 0, 1)), (10, 6, 2, (1, 2)), (2, 2, 0, (1,))])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_rows(dtype, d, dim, offset, sections, interleaved):
    g = torch.Generator().manual_seed(d + dim)
    n, hq, hk = 5, 7, 3
    q, k = (torch.randn(n, h, d, generator=g).to("cuda", dtype) for h in (hq, hk))
    pos = torch.randint(-2**31, 2**31 - 1, (len(sections), n), generator=g).int()
    pos[:, 0], pos[:, 1], pos[:, 2] = 0, 2**31 - 1, -2**31
    plan = ops.rotary_plan(d, rotary_dim=dim, offset=offset, sections=sections, interleaved=interleaved)
    p = (pos if len(sections) > 1 else pos[0]).cuda()
    for inverse in (False, True):
        a, b = ops.rotary(q, k, p, plan, inverse=inverse)
        assert a.shape == q.shape and b.shape == k.shape and a.is_contiguous() and a.dtype == dtype
        _check_rotary(q, a, pos.numpy(), plan, _freqs(dim), inverse)
        _check_rotary(k, b, pos.numpy(), plan, _freqs(dim), inverse)
    alone, none = ops.rotary(k, None, p, plan)
    assert none is None and torch.equal(alone, ops.rotary(q, k, p, plan)[1])


@pytest.mark.parametrize("batch,tokens", [(1, 1), (2, 3), (3, 700), (1, 2500)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotary_heads_of_any_strides(batch, tokens, dtype):
    """[B, T, H, d] becomes [B, H, T, d]; expanded positions and heads, rows that no wide word fits."""
    g = torch.Generator().manual_seed(tokens)
    plan = ops.rotary_plan(64, sections=(8, 24), interleaved=True, base=500.0)
    x = torch.randn(batch, tokens, 5, 64, generator=g).to("cuda", dtype)
    pos = torch.randint(0, 100000, (2, tokens), generator=g).int()
    p = pos.cuda().unsqueeze(1).expand(2, batch, tokens)
    want = ops.rotary(x.transpose(1, 2).contiguous(), None, p.contiguous(), plan)[0]
    some = slice(0, min(tokens, 9))
    _check_rotary(x[:, some], want.transpose(1, 2)[:, some], pos[:, None, some].expand(2, batch, -1).numpy(), plan, _freqs(64, 500.0))
    odd = torch.empty(batch * tokens * 5 * 67 + 1, dtype=dtype, device="cuda")[1:].view(batch, tokens, 5, 67)[..., 2:66]
    odd.copy_(x)
    fp = torch.empty(batch, 5, 64, tokens, dtype=dtype, device="cuda").permute(0, 1, 3, 2)  # (no unit stride along d)
    fp.copy_(x.transpose(1, 2))
    for view in (x.transpose(1, 2), odd.transpose(1, 2), fp):
        got, _ = ops.rotary(view, None, p, plan)
        assert got.is_contiguous() and torch.equal(got, want)
    one = x[:, :, :1].transpose(1, 2)
    shared, _ = ops.rotary(one.expand(batch, 5, tokens, 64), one, p, plan)
    assert torch.equal(shared, want[:, :1].expand(batch, 5, tokens, 64))


@pytest.mark.parametrize("hq,hkv", [(1, 0), (2, 1), (7, 1)])
@pytest.mark.parametrize("d,dim,offset,dtype", [(64, 64, 0, torch.bfloat16), (72, 36, 36, torch.float32), (128, 14, 2, torch.float16),
                                                (256, 256, 0, torch.bfloat16)])
def test_rotary_few_heads_and_many_tokens(hq, hkv, d, dim, offset, dtype):
    """Several tokens a block: bit for bit what calls of a few tokens give, with a last block that is not full."""
    g = torch.Generator(device="cuda").manual_seed(d + hq)
    plan = ops.rotary_plan(d, rotary_dim=dim, offset=offset, sections=(dim // 2 - 2, 2))
    for batch, tokens in [(1, 593), (3, 1999), (2, 9001)]:
        q, k = (torch.randn(batch, tokens, h, d, generator=g, device="cuda").to(dtype).transpose(1, 2) if h else None for h in (hq, hkv))
        pos = torch.randint(-2**31, 2**31 - 1, (2, batch, tokens), generator=g, device="cuda", dtype=torch.int32)
        got = ops.rotary(q, k, pos, plan)
        for b in range(batch):
            for t in range(0, tokens, 290):
                part = [None if x is None else x[b:b + 1, :, t:t + 290] for x in (q, k)]
                for x, y in zip(got, ops.rotary(*part, pos[:, b:b + 1, t:t + 290], plan)):
                    assert (x is None and y is None) or torch.equal(x[b:b + 1, :, t:t + 290], y)


def test_rotary_empty_and_refusals():
    plan, p = ops.rotary_plan(64), torch.zeros(0, **I32)
    q = torch.zeros(0, 4, 64, device="cuda")
    a, b = ops.rotary(q, q[:, :1], p, plan)
    assert a.shape == (0, 4, 64) and b.shape == (0, 1, 64)
    a, b = ops.rotary(torch.ones(3, 0, 64, device="cuda"), torch.ones(3, 2, 64, device="cuda"), torch.zeros(3, **I32), plan)
    assert a.shape == (3, 0, 64) and (b == 1).all()
    q, p = torch.zeros(3, 4, 64, device="cuda"), torch.zeros(3, **I32)
    two = ops.rotary_plan(64, sections=(16, 16))
    for args in ((q, q.half(), p, plan), (q, q[:2], p, plan), (q.double(), None, p, plan), (q, None, p[:2], plan), (q, None, p.long(), plan),
                 (q, None, p, two), (q, None, p.view(1, 3).expand(3, 3), two), (q[..., :32], None, p, plan), (q[0], None, p, plan),
                 (q, q.cpu(), p, plan), (q, None, p.cpu(), plan), (q, None, p, plan._replace(turns=plan.turns[:5])),
                 (q, None, p, plan._replace(axis=plan.axis + 1)), (q, None, p, plan._replace(offset=2))):
        with pytest.raises(RuntimeError):
            ops.rotary(*args)


@pytest.mark.parametrize("layout", ["rows", "heads", "tokens"])
def test_rotary_gradients(layout):
    """The turn is linear: the gradient is the turn back (formula), and f(x + h) - f(x) is the turned h (differences)."""
    g = torch.Generator().manual_seed(4)
    plan = ops.rotary_plan(24, rotary_dim=16, offset=4, sections=(3, 5))
    shape = (6, 3, 24) if layout == "rows" else (2, 3, 6, 24) if layout == "heads" else (2, 6, 3, 24)
    pos = torch.randint(0, 5000, (2, 6) if layout == "rows" else (2, 2, 6), generator=g).int().cuda()
    x = torch.randn(shape, generator=g).cuda().requires_grad_()
    y = torch.randn(shape, generator=g).cuda()[..., :, :].requires_grad_()
    view = (lambda t: t.transpose(1, 2)) if layout == "tokens" else (lambda t: t)
    a, b = ops.rotary(view(x), view(y), pos, plan)
    da, db = (torch.randn(a.shape, generator=g).cuda() for _ in range(2))
    dx, dy = torch.autograd.grad((a, b), (x, y), (da, db), retain_graph=True)
    assert dx.shape == x.shape and dx.is_contiguous()
    rows = (lambda t: t) if layout == "rows" else (lambda t: t.transpose(1, 2))
    back = dx if layout == "rows" else dx if layout == "tokens" else dx.transpose(1, 2)
    _check_rotary(rows(da), back, pos.cpu().numpy(), plan, _freqs(16), inverse=True)
    assert torch.equal(torch.autograd.grad(a, x, da, retain_graph=True)[0], dx)  # K's output has no gradient
    assert torch.equal(torch.autograd.grad(b, y, db, retain_graph=True)[0], dy)
    alone, none = ops.rotary(view(x), None, pos, plan)
    assert none is None and torch.equal(torch.autograd.grad(alone, x, da)[0], dx)
    assert not any(t.requires_grad for t in ops.rotary(view(x).detach(), view(y).detach(), pos, plan))
    left, right = ops.rotary(view(x).detach(), view(y), pos, plan)  # (a gradient of K alone)
    assert torch.equal(torch.autograd.grad((left.sum() + (right * db).sum()), y)[0], dy)
    # differences: <da, f(x + h) - f(x)> = <dx, h>, but for fp32's rounding of sums of 2 * 6 * 3 * 24 terms
    h = torch.randn(shape, generator=g).cuda()
    with torch.no_grad():
        moved = ops.rotary(view(x + h), None, pos, plan)[0].double() - a.double()
    left, right = (da.double() * moved).sum(), (dx.double() * h.double()).sum()
    # each of the outputs and of x + h is off by at most 8 half steps of the largest |a| + |b|, each product by da
    bound = 2.0**-24 * 30 * float(da.double().abs().sum()) * 2 * float((x.abs().max() + h.abs().max()))
    assert abs(float(left - right)) <= bound
    # a gradient of the gradient: with respect to da it is the turn itself
    da = da.requires_grad_()
    (dx,) = torch.autograd.grad(a, x, da, create_graph=True)
    (again,) = torch.autograd.grad(dx, da, x.detach())
    assert torch.equal(again, ops.rotary(view(x.detach()), None, pos, plan)[0])


def test_rotary_training_step_in_a_graph():
    """Projections, rotary positions of three axes, selected attention, backward: captured while an eager graph of the same
    tensors lives (leaves of their own: torch ties a leaf to the stream of the graph that it is in), and replayed with other
    inputs."""
    g = torch.Generator().manual_seed(8)
    T, hq, hk, d = 192, 16, 2, 128
    weights = (torch.randn(d * (hq + 2 * hk), 32, generator=g) / 6).cuda()
    x = torch.randn(1, T, 32, generator=g).cuda()
    plan = ops.rotary_plan(d, sections=(16, 24, 24), base=1e6)
    pos = torch.arange(T, **I32).view(1, 1, T).expand(3, 1, T)
    sel = torch.randint(0, 3, (1, hk, T, 3), generator=g).int().cuda()

    def loss():
        w = weights.detach().requires_grad_()
        qkv = (x @ w.T).to(torch.bfloat16).view(1, T, hq + 2 * hk, d)
        q, k = ops.rotary(qkv[:, :, :hq].transpose(1, 2), qkv[:, :, hq:hq + hk].transpose(1, 2), pos, plan)
        v = qkv[:, :, hq + hk:].transpose(1, 2).contiguous()
        return ops.SelectedAttention.apply(q, k, v, sel).float().square().mean(), w

    def gradient():
        value, w = loss()
        return torch.autograd.grad(value, w)[0]

    eager = loss()
    (want,) = torch.autograd.grad(*eager, retain_graph=True)
    assert torch.isfinite(want).all() and want.abs().sum() > 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gradient()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gradient()
    for step in range(2):
        if step:
            x.copy_(torch.randn(1, T, 32, generator=g))
            want = gradient()
        graph.replay()
        # (atomic sums of the attention's backward: the order of up to 192 fp32 terms differs; dK and dV are then rounded to bf16)
        assert float((got - want).abs().max()) <= 2.0**-7 * float(want.abs().max())
    del eager


# ------------------------------------------------------------------ block selection
DIMS = [(64, 64), (128, 128), (192, 128), (128, 64)]


def _records(x, d_v, dtype=torch.bfloat16):
    """Keys [P, Hkv, 64, d_qk] as records (V of zeros)."""
    code, byte = oc.quantise(x.to(dtype).double().numpy())
    p, h = x.shape[:2]
    parts = [(code[..., 0::2] + 16 * code[..., 1::2]).reshape(p, h, -1), byte.reshape(p, h, -1), np.zeros((p, h, 36 * d_v))]
    return np.concatenate(parts, -1).astype(np.uint8)


def _tables(lens, block, stride, rng, spare=2):
    need = [-(-oracle.completed(max(t, 0), block, stride) // 64) for t in lens]
    pages = np.full((len(lens), max(max(need), 1)), -1, np.int32)
    ids = rng.permutation(sum(need) + spare).astype(np.int32)
    at = 0
    for s, n in enumerate(need):
        pages[s, :n] = ids[at:at + n]
        at += n
    return pages, sum(need) + spare


def _check_select(q, cache, pages, lens, n_sel, l_prime=64, block=32, stride=16, cu=None):
    got = ops.cache_select(q.cuda(), torch.from_numpy(cache).cuda(), _t(pages), _t(lens), n_sel, l_prime, block, stride,
                           None if cu is None else _t(cu))
    want = oracle.select(q.double().numpy(), cache, pages, np.asarray(lens), n_sel, l_prime, block, stride,
                         None if cu is None else np.asarray(cu))
    assert got.shape == want.shape and got.dtype == torch.int32
    bad = np.argwhere(got.cpu().numpy() != want)
    assert bad.size == 0, (bad[:4], got.cpu().numpy()[tuple(bad[0][:2])], want[tuple(bad[0][:2])])
    return want


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,n_sel,l_prime", [(16, 1, 16, 64), (8, 8, 3, 128), (14, 2, 40, 64), (5, 1, 1, 256)])
def test_select(dims, dtype, hq, hkv, n_sel, l_prime):
    rng = np.random.default_rng(dims[0] + hq)
    g = torch.Generator().manual_seed(dims[0] + hq + n_sel)
    lens = [1, 31, 32, 63, 64, 65, 1055, 2000, 5003, 0]
    pages, count = _tables(lens, 32, 16, rng)
    x = torch.randn(count, hkv, 64, dims[0], generator=g) * torch.exp(0.5 * torch.randn(dims[0], generator=g)) + 0.3
    q = torch.randn(len(lens), hq, dims[0], generator=g).to(dtype)
    want = _check_select(q, _records(x, dims[1], dtype), pages, lens, n_sel, l_prime)
    assert (want[-1] == -1).all() and (want[0, :, 0] == 0).all()


@pytest.mark.parametrize("block,stride,l_prime", [(1, 1, 64), (1, 1, 256), (16, 8, 128), (64, 64, 64), (7, 3, 64), (32, 512, 64)])
def test_select_other_compressions(block, stride, l_prime):
    rng, g = np.random.default_rng(block), torch.Generator().manual_seed(stride)
    lens = [block - 1, block, 700, 1500]
    pages, count = _tables(lens, block, stride, rng)
    cache = _records(torch.randn(count, 2, 64, 64, generator=g), 64)
    q = torch.randn(4, 6, 64, generator=g).to(torch.bfloat16)
    for n_sel in (1, 7, 64):
        _check_select(q, cache, pages, lens, n_sel, l_prime, block, stride)


def test_select_packed_rows():
    """Several rows a sequence, none, rows before the first and behind the last; more rows than a sequence has tokens."""
    rng, g = np.random.default_rng(3), torch.Generator().manual_seed(3)
    lens, cu = [900, 4, 0, 3000, 1700], [2, 6, 12, 13, 13, 21]
    pages, count = _tables(lens, 32, 16, rng)
    cache = _records(torch.randn(count, 3, 64, 128, generator=g), 128)
    q = torch.randn(24, 12, 128, generator=g).to(torch.float16)
    want = _check_select(q, cache, pages, lens, 9, 128, cu=cu)
    assert (want[:2] == -1).all() and (want[21:] == -1).all() and (want[6:8] == -1).all() and (want[8:12, :, 0] == 0).all()


def test_select_ties_go_to_the_lowest_block():
    """All keys alike, all zero, a query of zeros, two values only: hundreds of equal scores."""
    g = torch.Generator().manual_seed(5)
    lens = [20000, 3000]
    pages, count = _tables(lens, 32, 16, np.random.default_rng(5))
    same = torch.randn(1, 1, 1, 64, generator=g).expand(count, 1, 64, 64)
    two = same * torch.where(torch.rand(count, 1, 64, 1, generator=g) < 0.5, 1.0, -1.0)
    q = torch.randn(2, 4, 64, generator=g).to(torch.bfloat16)
    for x in (same, torch.zeros_like(same), two):
        for n_sel in (16, 300):
            _check_select(q, _records(x, 64), pages, lens, n_sel)
            _check_select(torch.zeros_like(q), _records(x, 64), pages, lens, n_sel)
    # (the first block has a key more than most, so that only it stands out)
    assert ops.cache_select(torch.zeros_like(q).cuda(), torch.from_numpy(_records(same, 64)).cuda(), _t(pages), _t(lens), 5)[0, 0].tolist() == [0, 1, 2, 3, 4]


def test_select_tells_close_scores_apart():
    """Blocks whose scores differ by 2^-36 of their size, which fp32 sums lose: one code of a tiny scale each."""
    g = torch.Generator().manual_seed(6)
    lens = [16 * 64 * 3 + 16]  # 193 keys
    pages, count = _tables(lens, 32, 16, np.random.default_rng(6))
    x = torch.randn(1, 1, 1, 128, generator=g).expand(count, 1, 64, 128).clone()
    x[..., :16] = 0
    step = torch.randperm(count * 64, generator=g).view(count, 64) % 8
    x[:, 0, :, 0] = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])[step] * 2.0**-13
    x[:, 0, :, 1] = 6 * 2.0**-13
    q = torch.randn(1, 16, 128, generator=g) * 2.0**6
    q[..., 0] = 2.0**-15
    want = _check_select(q.to(torch.bfloat16), _records(x, 128), pages, lens, 32)
    assert sorted(want[0, 0].tolist()) != want[0, 0].tolist()


def test_select_of_what_is_no_number():
    """Keys of NaN and infinity rank last, a query with one ranks nothing (the lowest blocks); missing pages count as zeros."""
    g = torch.Generator().manual_seed(7)
    lens = [4000, 4000, 4000]
    pages, count = _tables(lens, 32, 16, np.random.default_rng(7))
    x = torch.randn(count, 2, 64, 64, generator=g)
    x[pages[0, 1], 0, 5, 3], x[pages[0, 0], 1, 60, 0] = math.nan, math.inf
    x[pages[1, 2], 0] = math.nan
    cache = _records(x, 64)
    q = torch.randn(3, 8, 64, generator=g).to(torch.bfloat16)
    q[2, 1, 5], q[2, 7, 0] = math.inf, -math.inf
    want = _check_select(q, cache, pages, lens, 16)
    assert want[2, 0].tolist() == list(range(16))
    _check_select(q, cache, pages, lens, 100)
    pages[0, 1], pages[1, 0], pages[1, 2] = -1, count, -2**31
    _check_select(q, cache, pages, lens, 16)
    for lens in ([-5, 2**31 - 1, 4096 + 32], [4095 + 32, 4095 + 31, 70]):
        _check_select(q, cache, pages, lens, 8)


def test_select_takes_scores_of_any_size():
    """A block that stands out a million times, tiny and huge queries, scales from the smallest to the largest."""
    g = torch.Generator().manual_seed(8)
    lens = [9000] * 4
    pages, count = _tables(lens, 32, 16, np.random.default_rng(8))
    x = torch.randn(count, 1, 64, 64, generator=g) * torch.exp2(torch.randint(-17, 13, (count, 1, 64, 4, 1), generator=g).float()).expand(
        -1, -1, -1, -1, 16).reshape(count, 1, 64, 64)
    cache = _records(x.clamp(-50000, 50000), 64)
    for scale in (1.0, 2.0**-120, 2.0**100):
        q = (torch.randn(4, 3, 64, generator=g) * scale).to(torch.bfloat16)
        _check_select(q, cache, pages, lens, 24)
    x = torch.randn(count, 1, 64, 64, generator=g) * 2.0**-6
    x[pages[0, 0], 0, 1] = 2.0**14
    q = torch.randn(4, 3, 64, generator=g).to(torch.float16)
    _check_select(q, _records(x, 64), pages, lens, 24)


def test_select_most_blocks_and_heads():
    """1024 blocks of more than there are, 256 query heads for a KV head, more rows than a launch takes."""
    g = torch.Generator().manual_seed(9)
    lens = [70000, 40]
    pages, count = _tables(lens, 32, 16, np.random.default_rng(9))
    cache = _records(torch.randn(count, 1, 64, 64, generator=g), 64)
    _check_select(torch.randn(2, 256, 64, generator=g).to(torch.bfloat16), cache, pages, lens, 1024)
    rows = 2300
    lens = np.random.default_rng(2).integers(0, 700, rows)
    pages = np.random.default_rng(3).integers(0, count, (rows, 1)).astype(np.int32)
    _check_select(torch.randn(rows, 2, 64, generator=g).to(torch.bfloat16), cache, pages, lens, 6)


@pytest.mark.parametrize("dims", DIMS[:3])
@pytest.mark.parametrize("hq,n_sel,l_prime", [(8, 16, 64), (24, 700, 64), (40, 5, 128)])
def test_select_of_many_rows(dims, hq, n_sel, l_prime):
    """More rows and KV heads than fit the GPU at once, up to 1024 blocks a row, of them equal ones and some of no number."""
    rng, g = np.random.default_rng(dims[0] + hq), torch.Generator().manual_seed(dims[0] + hq)
    lens = np.concatenate([rng.integers(0, 3000, 127), [65536 if l_prime == 64 else 40001, 0]])
    pages, count = _tables(lens[-2:], 32, 16, rng)
    pages = np.stack([np.roll(pages[0], r) for r in range(len(lens))])
    x = torch.randn(count, 8, 64, dims[0], generator=g)
    x[:, 6] = x[:1, 6, :1]
    x[1, 7, 5, 3] = math.nan
    q = torch.randn(len(lens), hq, dims[0], generator=g).to(torch.bfloat16)
    q[3, 0, 0] = math.inf
    _check_select(q, _records(x, dims[1]), pages, lens, n_sel, l_prime)


def test_select_of_many_rows_whose_last_block_has_no_page():
    """1024 blocks of whole pages and the tokens behind them, which the last compressed key covers, in one block more."""
    rng, g = np.random.default_rng(12), torch.Generator().manual_seed(12)
    lens = np.concatenate([[65567, 65537, 65568, 65536], rng.integers(0, 900, 200)])
    pages, count = _tables([65536], 32, 16, rng)
    pages = np.repeat(pages, len(lens), 0)
    assert pages.shape[1] == 64
    cache = _records(torch.randn(count, 4, 64, 64, generator=g), 64)
    q = torch.randn(len(lens), 4, 64, generator=g).to(torch.float16)
    for n_sel in (16, 600):
        want = _check_select(q, cache, pages, lens, n_sel)
        assert (want[:2, :, :n_sel] >= 0).all() and (want[2] == -1).all()


def test_select_strides_streams_and_refusals():
    g = torch.Generator().manual_seed(10)
    lens = [3000, 2500]
    pages, count = _tables(lens, 32, 16, np.random.default_rng(10))
    cache = torch.from_numpy(_records(torch.randn(count, 2, 64, 128, generator=g), 64)).cuda()
    q = torch.randn(2, 8, 128, generator=g).to(torch.bfloat16).cuda()
    p, n = _t(pages), _t(lens)
    want = ops.cache_select(q, cache, p, n, 12)
    wide = torch.zeros(2, 9, 160, dtype=q.dtype, device="cuda")
    wide[:, :8, 16:144] = q
    assert torch.equal(ops.cache_select(wide[:, :8, 16:144], cache, p, n, 12), want)
    one = ops.cache_select(q[:1].expand(2, 8, 128), cache, p, n, 12)
    assert torch.equal(one[0], want[0])
    big = torch.zeros(count, 3, cache.shape[2], dtype=torch.uint8, device="cuda")
    big[:, :2] = cache
    table = torch.full((2, p.shape[1] + 5), 3, **I32)
    table[:, :p.shape[1]] = p
    assert torch.equal(ops.cache_select(q, big[:, :2], table[:, :p.shape[1]], n, 12), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        twice = [ops.cache_select(q, cache, p, n, 12) for _ in range(3)]
    here = [ops.cache_select(q, cache, p, n, 12) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in twice + here)
    for bad in (dict(n_sel=0), dict(n_sel=1025), dict(l_prime=96), dict(cmp_block=0), dict(cmp_stride=0), dict(Q=q.float()), dict(Q=q[:, :7]),
                dict(Q=q[..., 1:65]), dict(lens=n[:1]), dict(cmp_pages=p.long()), dict(cu_seqlens=n), dict(Q=q.cpu())):
        with pytest.raises(RuntimeError):
            ops.cache_select(**{**dict(Q=q, cmp_cache=cache, cmp_pages=p, lens=n, n_sel=12), **bad})


# ------------------------------------------------------------------ whole steps
@pytest.mark.parametrize("captured", [False, True])
def test_decode_steps_from_request_lengths(captured):
    """Requests come, get tokens one by one and end: pages, rotary positions, both caches, selection and the three branches of
    every step, and each token's results against those of a sequence that is computed by itself."""
    g = torch.Generator().manual_seed(21)
    S, hq, hk, d, width, n_sel = 4, 8, 2, 64, 4, 2
    plan = ops.rotary_plan(d, sections=(8, 12, 12))
    cache, cmp_cache = ops.cache_alloc(S * width, hk, d, d), ops.cache_alloc(S, hk, d, d)
    state = [torch.full((S, width), -1, **I32), torch.zeros(S, **I32), torch.zeros(S, **I32), torch.randperm(S * width, generator=g).int().cuda(),
             _t([S * width])]
    cmp_pages = torch.arange(S, **I32).flip(0).view(S, 1).contiguous()
    q, k, v = (torch.randn(S, h, d, generator=g).to("cuda", torch.bfloat16) for h in (hq, hk, hk))

    def step():
        batch = ops.cache_reserve(*state)
        a, b = ops.rotary(q, k, batch.positions.expand(3, S), plan)
        ops.cache_write(cache, b, v, state[0], batch.lens)
        cmp_lens = nsa.cache_compress(cache, d, state[0], batch.lens, cmp_cache, cmp_pages)
        out = nsa.nsa_decode(a, cache, state[0], batch.lens, l_prime=64, window=32, cmp_cache=cmp_cache, cmp_pages=cmp_pages,
                             cmp_lens=cmp_lens, n_sel=n_sel)
        return out, batch, ops.cache_select(a, cmp_cache, cmp_pages, batch.lens, n_sel)

    # prompts of the first requests, in one packed call
    prompt = [70, 200, 0, 131]
    state[2].copy_(_t(prompt))
    total = sum(prompt)
    batch = ops.cache_reserve(*state, n_tokens=total)
    assert torch.equal(batch.positions, torch.cat([torch.arange(n, **I32) for n in prompt]))
    history = [[] for _ in range(S)]
    pk, pv = (torch.randn(total, hk, d, generator=g).to("cuda", torch.bfloat16) for _ in range(2))
    _, rk = ops.rotary(pk.new_zeros(total, 1, d), pk, batch.positions.expand(3, total), plan)
    ops.cache_write(cache, rk, pv, state[0], batch.lens, cu_seqlens=batch.cu_seqlens)
    nsa.cache_compress(cache, d, state[0], batch.lens, cmp_cache, cmp_pages, cu_seqlens=batch.cu_seqlens, n_tokens=total)
    at = np.cumsum([0] + prompt)
    for s in range(S):
        history[s] = [(pk[i], pv[i]) for i in range(at[s], at[s + 1])]
    state[2].copy_(_t([1, 1, 0, 1]))
    graph, outs = torch.cuda.CUDAGraph(), None
    if captured:
        saved = [t.clone() for t in state] + [cache.clone(), cmp_cache.clone()]
        step()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            outs = step()
        for t, old in zip(state + [cache, cmp_cache], saved):
            t.copy_(old)
    for i in range(6):
        rows = [1, -len(history[1]) if i == 2 else 0 if i in (3, 4) else 1, 1 if i > 2 else 0, 1 if i != 4 else 0]
        if i == 5:
            rows[1] = 1  # (a new request where the ended one was)
        state[2].copy_(_t(rows))
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        for s in range(S):
            history[s] = history[s] + [(k[s].clone(), v[s].clone())] if rows[s] > 0 else [] if rows[s] < 0 else history[s]
        if captured:
            graph.replay()
        out, batch, sel = outs if captured else step()
        assert batch.held.tolist() == [len(x) for x in history] == state[1].tolist()
        for s in range(S):
            if rows[s] <= 0:
                assert int(batch.lens[s]) == 0 and (out[s] == 0).all() and (sel[s] == -1).all()
                continue
            # the sequence by itself, in a cache of its own, written at once
            n = len(history[s])
            one, small = ops.cache_alloc(width, hk, d, d), ops.cache_alloc(1, hk, d, d)
            pages, lens, cu = torch.arange(width, **I32).view(1, width), _t([n]), _t([0, n])
            kk, vv = (torch.stack([x[j] for x in history[s]]) for j in range(2))
            pos = torch.arange(n, **I32)
            _, kk = ops.rotary(kk[:, :1], kk, pos.expand(3, n), plan)
            ops.cache_write(one, kk, vv, pages, lens, cu_seqlens=cu)
            cmp_lens = nsa.cache_compress(one, d, pages, lens, small, pages[:, :1], cu_seqlens=cu, n_tokens=n)
            a, _ = ops.rotary(q[s:s + 1], None, pos[-1:].expand(3, 1), plan)
            best = oracle.select(a.double().cpu().numpy(), small.cpu().numpy(), np.zeros((1, 1), np.int32), np.array([n]), n_sel)
            assert np.array_equal(sel[s].cpu(), best[0])
            want = nsa.nsa_decode(a, one, pages, lens, _t(best), window=32, cmp_cache=small, cmp_pages=pages[:, :1], cmp_lens=cmp_lens)
            # (the same values and keys; only how the attention shares out a batch's rows, and so its fp32 sums, may differ:
            # the bound of the attention's own tests is far above 2^-10 of the largest |v|)
            assert float((out[s] - want[0]).abs().max()) <= 2.0**-10 * float(vv.float().abs().max())
