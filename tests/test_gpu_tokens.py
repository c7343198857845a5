"""Tokens sorted by expert and back (permute, combine) and their gradients, against their definitions
in 64 bits.

Bounds.  u = finfo(dtype).eps / 2 is the relative error of one rounding, v = 2^-24 that of fp32.  A sum
of n fp32 products accumulated in any order is off by at most (n + 1) v sum|terms| (n roundings of
products, fewer with fused multiply-adds, and n - 1 of sums, to first order); the store rounds once more:
u (|exact| + that error), or half a subnormal step where the result is tiny.
"""

import numpy as np
import pytest
import torch

from vybforge_b200 import _lib, moe

pytestmark = pytest.mark.gpu
V = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def make_ids(T, k, E, mode, seed):
    rng = np.random.default_rng(seed)
    if mode == "repeat":                      # a token may name one expert on several lanes
        return rng.integers(0, E, (T, k)).astype(np.int32)
    idx = np.argsort(rng.random((T, max(E, k))), axis=1)[:, :k].astype(np.int32) % E
    if mode == "dropped":                     # negative and too large ids carry no row
        m = rng.random((T, k))
        idx[m < 0.2] = -1
        idx[m > 0.9] = E + rng.integers(0, 3)
        if T > 2:
            idx[1] = -7                       # a padded token: no row at all
    elif mode == "none":
        idx[:] = -1
    elif mode == "one":                       # every lane names the last expert
        idx[:] = E - 1
    return idx


def order(idx, E):
    """(perm_tok, pos_of, offsets) of the kept lanes by (expert, token, lane)."""
    T, k = idx.shape
    flat = idx.reshape(-1).astype(np.int64)
    kept = np.flatnonzero((flat >= 0) & (flat < E))
    lanes = kept[np.argsort(flat[kept], kind="stable")]
    pos = np.full(T * k, -1, np.int64)
    pos[lanes] = np.arange(len(lanes))
    perm = np.full(T * k, -1, np.int64)
    perm[:len(lanes)] = lanes // k
    off = np.concatenate([[0], np.cumsum(np.bincount(flat[kept], minlength=E))])
    return perm, pos, off


def within(got, want, err, dtype):
    """|got - want| <= err + one rounding to dtype; both on the GPU in fp64."""
    info = torch.finfo(dtype)
    tol = err + info.eps / 2 * (want.abs() + err) + info.smallest_normal * info.eps / 2
    d = (got.double() - want).abs()
    assert bool((d <= tol).all()), f"worst {float((d / tol).max()):.3g} of the bound"


SHAPES = [(1, 8, 256, 6144), (1, 1, 1, 1), (2, 2, 3, 7), (33, 4, 16, 1024), (257, 7, 64, 1023), (64, 32, 33, 200),
          (513, 4, 16, 72), (300, 8, 1000, 129), (1100, 32, 1024, 40), (5000, 3, 5, 8), (2049, 1, 97, 264)]


@pytest.mark.parametrize("mode", ["plain", "dropped", "repeat", "none", "one"])
@pytest.mark.parametrize("T,k,E,H", SHAPES)
def test_permute_is_the_stable_order(T, k, E, H, mode):
    dtype = DTYPES[(T + H) % 3]
    idx = make_ids(T, k, E, mode, seed=T + k)
    perm, pos, off = order(idx, E)
    x = torch.randn(T, H, device="cuda").to(dtype)
    out = torch.full((T * k, H), 7.0, dtype=dtype, device="cuda")
    xs, plan = moe.permute(x, torch.from_numpy(idx).cuda(), E, out=out)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(plan.pos_of.cpu().numpy(), pos)
    np.testing.assert_array_equal(plan.perm_tok.cpu().numpy(), perm)
    np.testing.assert_array_equal(plan.offsets.cpu().numpy(), off)
    np.testing.assert_array_equal(plan.counts.cpu().numpy(), np.diff(off))
    n = int(off[-1])
    assert torch.equal(xs[:n], x[torch.from_numpy(perm[:n]).cuda()])
    assert bool((xs[n:] == 7.0).all())        # rows behind the last one stay as they were
    none, again = moe.permute(None, torch.from_numpy(idx).cuda(), E)
    assert none is None and all(torch.equal(a, b) for a, b in zip(plan, again))


@pytest.mark.parametrize("E", [1, 5, 256, 1024])
@pytest.mark.parametrize("T,k,skew", [(8193, 8, 0.0), (8192, 8, 1.1), (32769, 8, 1.1), (131072, 2, 0.0), (70001, 1, 1.1)])
def test_plans_of_many_lanes(T, k, skew, E):
    """Above 65,536 lanes a warp's run of ids no longer fits its registers and is read in several passes; ids skewed towards a
    few experts, repeated within a token, dropped on both sides of the range."""
    rng = np.random.default_rng(T + E)
    p = np.arange(1, E + 1) ** -skew
    idx = rng.choice(rng.permutation(E), size=(T, k), p=p / p.sum()).astype(np.int32)
    m = rng.random((T, k))
    idx[m < 0.1] = -1
    idx[m > 0.95] = E + 1
    perm, pos, off = order(idx, E)
    none, plan = moe.permute(None, torch.from_numpy(idx).cuda(), E)
    x = torch.randn(T, 8, device="cuda").half()
    xs, again = moe.permute(x, torch.from_numpy(idx).cuda(), E)
    for got in (plan, again):
        np.testing.assert_array_equal(got.pos_of.cpu().numpy(), pos)
        np.testing.assert_array_equal(got.perm_tok.cpu().numpy(), perm)
        np.testing.assert_array_equal(got.offsets.cpu().numpy(), off)
        np.testing.assert_array_equal(got.counts.cpu().numpy(), np.diff(off))
    n = int(off[-1])
    assert torch.equal(xs[:n], x[torch.from_numpy(perm[:n]).cuda()])


@pytest.mark.parametrize("T,k,E", [(37, 4, 16), (700, 8, 64)])
def test_permute_plan_is_that_of_dispatch(T, k, E):
    idx = torch.from_numpy(make_ids(T, k, E, "plain", seed=3)).cuda()
    _, plan = moe.permute(None, idx, E)
    for a, b in zip(plan, moe.dispatch(idx, E)):
        assert torch.equal(a, b)


def rows_case(T, k, E, H, dtype, mode, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    idx = make_ids(T, k, E, mode, seed)
    _, pos, off = order(idx, E)
    y = torch.randn(T * k, H, device="cuda", generator=g).to(dtype)
    y[int(off[-1]):] = float("nan")           # rows that no lane names are never read
    w = torch.rand(T, k, device="cuda", generator=g)
    pos_t = torch.from_numpy(pos.astype(np.int32)).cuda()
    w.view(-1)[pos_t < 0] = float("nan")      # nor are the weights of dropped lanes
    return idx, pos_t, int(off[-1]), y, w, g


def gathered(y, pos, T, k):
    """fp64 [T, k, H] rows of the lanes, zero where dropped, and the kept mask [T, k, 1]."""
    kept = (pos >= 0).view(T, k, 1)
    return torch.where(kept, y.double()[pos.clamp(min=0).long()].view(T, k, -1), 0.0), kept


@pytest.mark.parametrize("mode", ["plain", "dropped", "none"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,H", SHAPES[:9])
def test_permute_backward(T, k, E, H, dtype, mode):
    _, pos, n, y, _, _ = rows_case(T, k, E, H, dtype, mode, seed=11)
    v, _ = gathered(y, pos, T, k)
    for out in (None, torch.float32, torch.bfloat16):
        dx = moe.permute_backward(y, pos, T, k, out_dtype=out)
        assert dx.dtype == (out or dtype)
        within(dx, v.sum(1), (k + 1) * V * v.abs().sum(1), dx.dtype)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("mode", ["plain", "dropped"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,H", SHAPES[:9])
def test_combine_any_type_and_length(T, k, E, H, dtype, mode, shared):
    _, pos, n, y, w, g = rows_case(T, k, E, H, dtype, mode, seed=12)
    v, kept = gathered(y, pos, T, k)
    t = torch.where(kept, v * w.double().view(T, k, 1), 0.0)
    ys = torch.randn(T, H, device="cuda", generator=g).to(dtype) if shared else None
    want, size = t.sum(1), t.abs().sum(1)
    if shared:
        want, size = want + ys.double(), size + ys.double().abs()
    for out in DTYPES:
        got = moe.combine(y, pos, w, T, k, y_shared=ys, out_dtype=out)
        within(got, want, (k + 2) * V * size, out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,H", [(1, 8, 6144), (32, 6, 6144), (260, 8, 1020), (260, 3, 1028), (130, 6, 2052), (300, 16, 1024),
                                   (64, 9, 4096), (2050, 2, 132), (1040, 5, 264), (5, 2, 70000)])
def test_words_of_every_width_give_the_same_bits(T, k, H, dtype):
    """Row lengths and counts on both sides of each rule that chooses 16-byte words, 8-byte words, columns or the
    layer's kernel: the values are those of the definition, and the bits those of the element path."""
    _, pos, n, y, w, g = rows_case(T, k, 16, H, dtype, "dropped", seed=14)
    v, kept = gathered(y, pos, T, k)
    t = torch.where(kept, v * w.double().view(T, k, 1), 0.0)
    ys = torch.randn(T, H, device="cuda", generator=g).to(dtype)
    y1 = torch.empty(y.numel() + 1, dtype=dtype, device="cuda")[1:].view(y.shape).copy_(y)   # no word begins at its address
    for shared in (None, ys):
        want, size = t.sum(1), t.abs().sum(1)
        if shared is not None:
            want, size = want + ys.double(), size + ys.double().abs()
        for out in DTYPES:
            got = moe.combine(y, pos, w, T, k, y_shared=shared, out_dtype=out)
            within(got, want, (k + 2) * V * size, out)
            assert torch.equal(got, moe.combine(y1, pos, w, T, k, y_shared=shared, out_dtype=out))
    assert torch.equal(moe.permute_backward(y, pos, T, k), moe.permute_backward(y1, pos, T, k))


def test_combine_takes_longer_buffers_and_more_tokens():
    """Buffers with room for more tokens than the call has (the positions, the weights and the shared rows), and more
    lanes than a sorted plan may have: 2^27 + 1 tokens of 8 lanes, almost all without a row."""
    g = torch.Generator(device="cuda").manual_seed(15)
    T, k, H, room = 5, 2, 64, 9
    y = torch.randn(room * k, H, device="cuda", generator=g)
    pos = torch.randperm(room * k, device="cuda", generator=g).int()
    w = torch.rand(room, k, device="cuda", generator=g)
    ys = torch.randn(room, H, device="cuda", generator=g)
    whole = moe.combine(y, pos, w, room, k, y_shared=ys, out_dtype=torch.float32)
    assert torch.equal(moe.combine(y, pos, w, T, k, y_shared=ys, out_dtype=torch.float32), whole[:T])
    assert torch.equal(moe.combine(y, pos, w, T, k, y_shared=ys.view(1, room, H), out_dtype=torch.float32), whole[:T])
    with pytest.raises(_lib.VfmoeError):
        moe.combine(y, pos, w, T, k, y_shared=ys[:T - 1])
    T, k, H = (1 << 27) + 1, 8, 4
    y = torch.randn(16, H, device="cuda", generator=g).half()
    pos = torch.full((T * k,), -1, dtype=torch.int32, device="cuda")
    pos[:8] = torch.arange(8, dtype=torch.int32, device="cuda")
    pos[-8:] = torch.arange(8, 16, dtype=torch.int32, device="cuda")
    out = moe.combine(y, pos, None, T, k, out_dtype=torch.float16)
    v = y.double().view(2, 8, H)
    within(out[[0, T - 1]], v.sum(1), (k + 2) * V * v.abs().sum(1), torch.float16)
    assert int(out.count_nonzero()) <= 2 * H


@pytest.mark.parametrize("mode", ["plain", "dropped", "none"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,H", SHAPES[:9])
def test_combine_backward(T, k, E, H, dtype, mode):
    _, pos, n, y, w, g = rows_case(T, k, E, H, dtype, mode, seed=13)
    v, kept = gathered(y, pos, T, k)
    for gt in (dtype, torch.float32):
        dout = torch.randn(T, H, device="cuda", generator=g).to(gt)
        d = dout.double().unsqueeze(1)
        dy0 = torch.full_like(y, 5.0)
        dy, dw = moe.combine_backward(dout, y, pos, w, T, k, dy=dy0)
        assert dy.data_ptr() == dy0.data_ptr() and bool((dy[n:] == 5.0).all())
        lanes = (pos >= 0).nonzero().squeeze(1)
        want = (d * w.double().unsqueeze(-1)).view(T * k, H)[lanes]
        within(dy[pos[lanes].long()], want, V * want.abs(), dtype)
        within(dw, torch.where(kept, d * v, 0.0).sum(-1), (H + 1) * V * (d * v).abs().sum(-1), torch.float32)
        # weight 1 where no weights are given
        dy1, dw1 = moe.combine_backward(dout, y, pos, None, T, k)
        within(dy1[pos[lanes].long()], d.expand(T, k, H).reshape(T * k, H)[lanes], torch.zeros((), device="cuda"),
               dtype)
        assert torch.equal(dw1, dw)
        # in place of the rows
        y2 = y.clone()
        dy2, dw2 = moe.combine_backward(dout, y2, pos, w, T, k, dy=y2)
        assert torch.equal(dy2[:n], dy[:n]) and torch.equal(dw2, dw)


def test_gradients_against_differences():
    """d<out, r>/dparameter by central differences in 64 bits of the composed map x -> permute -> 2x -> combine."""
    T, k, E, H = 5, 3, 7, 16
    idx = make_ids(T, k, E, "dropped", seed=4)
    perm, pos, off = order(idx, E)
    pos_t = torch.from_numpy(pos.astype(np.int32)).cuda()
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(T, H, device="cuda", generator=g)
    w = torch.rand(T, k, device="cuda", generator=g)
    r = torch.randn(T, H, device="cuda", generator=g)
    kept = (pos_t >= 0).view(T, k)

    def f(xv, wv):
        return ((torch.where(kept, wv, 0.0).unsqueeze(-1) * 2.0 * xv.unsqueeze(1)).sum(1) * r.double()).sum()

    xs, plan = moe.permute(x, torch.from_numpy(idx).cuda(), E)
    n = int(off[-1])
    y = torch.zeros_like(xs)
    y[:n] = 2.0 * xs[:n]
    dy, dw = moe.combine_backward(r, y, plan.pos_of, w, T, k)
    dx = moe.permute_backward(2.0 * dy, plan.pos_of, T, k)
    h = 1e-4
    for got, which in ((dx, 0), (dw, 1)):
        base = [x.double(), w.double()]
        flat = got.reshape(-1).double()
        for i in range(flat.numel()):
            up, dn = [b.clone() for b in base], [b.clone() for b in base]
            up[which].view(-1)[i] += h
            dn[which].view(-1)[i] -= h
            diff = float(f(*up) - f(*dn)) / (2 * h)    # f is linear in each: no truncation error
            # fp32 sums of at most H terms of size |2 x r| < 50, and the cancellation 1e-16 * |f| / h of diff
            assert abs(float(flat[i]) - diff) <= (H + 2) * V * 50 * H + 1e-9, (which, i)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_at_odd_addresses(dtype):
    """Views that start one element into their storage take the element path and give the same rows."""
    T, k, E, H = 40, 4, 16, 64
    idx = torch.from_numpy(make_ids(T, k, E, "plain", seed=6)).cuda()
    x = torch.randn(T, H, device="cuda").to(dtype)

    def shifted(t):
        s = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
        return s.copy_(t)

    xs, plan = moe.permute(x, idx, E)
    xs1, _ = moe.permute(shifted(x), idx, E, out=shifted(torch.zeros_like(xs)))
    assert torch.equal(xs, xs1)
    w = torch.rand(T, k, device="cuda")
    assert torch.equal(moe.combine(xs, plan.pos_of, w, T, k, out_dtype=dtype),
                       moe.combine(shifted(xs), plan.pos_of, w, T, k, out_dtype=dtype))
    dout = torch.randn(T, H, device="cuda").to(dtype)
    dy, dw = moe.combine_backward(dout, xs, plan.pos_of, w, T, k)
    dy1, dw1 = moe.combine_backward(shifted(dout), shifted(xs), plan.pos_of, w, T, k, dy=shifted(xs))
    assert torch.equal(dy, dy1)
    # the element path adds the same products in another order
    within(dw1, dw.double(), 2 * (H + 1) * V * (dout.double().abs().sum(1, keepdim=True) * xs.double().abs().max()),
           torch.float32)


def test_offsets_beyond_32_bits():
    """400,000 rows of 6,144: row addresses pass 2^31 elements."""
    T, k, E, H = 50000, 8, 256, 6144
    idx = torch.randint(0, E, (T, k), dtype=torch.int32, device="cuda")
    x = torch.randn(T, H, device="cuda", dtype=torch.bfloat16)
    xs, plan = moe.permute(x, idx, E)
    pick = torch.randint(0, T * k, (4096,), device="cuda")
    pick[0], pick[1] = 0, T * k - 1
    assert torch.equal(xs[pick], x[plan.perm_tok[pick].long()])
    dx = moe.permute_backward(xs, plan.pos_of, T, k)
    toks = torch.arange(T - 2000, T, device="cuda")
    assert torch.equal(dx[toks], (8.0 * x[toks].float()).to(torch.bfloat16))  # 8 equal rows: exact
    w = torch.ones(T, k, device="cuda")
    dy, dw = moe.combine_backward(x, xs, plan.pos_of, w, T, k, dy=xs)          # in place
    assert torch.equal(dy[pick], x[plan.perm_tok[pick].long()])
    n2 = x[toks].double().square().sum(1, keepdim=True).expand(-1, k)
    within(dw[toks], n2, (H + 1) * V * n2, torch.float32)


def test_no_tokens():
    idx = torch.empty((0, 4), dtype=torch.int32, device="cuda")
    xs, plan = moe.permute(torch.empty((0, 64), device="cuda"), idx, 16)
    assert xs.shape == (0, 64) and int(plan.offsets.abs().sum()) == 0 and int(plan.counts.abs().sum()) == 0
    assert moe.permute_backward(xs, plan.pos_of, 0, 4).shape == (0, 64)
    dy, dw = moe.combine_backward(xs, xs, plan.pos_of, None, 0, 4)
    assert dy.shape == (0, 64) and dw.shape == (0, 4)


@pytest.mark.parametrize("T", [16, 600])
def test_captured_with_new_ids_on_another_stream(T):
    """One captured graph of the way out, back and its gradients, replayed on other ids and rows; two
    graphs alive at once share nothing."""
    k, E, H = 8, 32, 256
    graphs = []
    for s in range(2):
        x = torch.zeros(T, H, device="cuda", dtype=torch.bfloat16)
        idx = torch.zeros(T, k, dtype=torch.int32, device="cuda")
        w = torch.rand(T, k, device="cuda")

        def step(x=x, idx=idx, w=w):
            xs, plan = moe.permute(x, idx, E)
            out = moe.combine(xs, plan.pos_of, w, T, k)
            dy, dw = moe.combine_backward(x, xs, plan.pos_of, w, T, k)
            return xs, out, dy, dw, moe.permute_backward(dy, plan.pos_of, T, k)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                res = step()
        graphs.append((gr, x, idx, step, res))
    torch.cuda.synchronize()
    for gr, x, idx, _, _ in graphs:
        x.copy_(torch.randn_like(x))
        idx.copy_(torch.randint(0, E, idx.shape, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        for s, g in zip((s1, s2), graphs):
            with torch.cuda.stream(s):
                g[0].replay()
    torch.cuda.synchronize()
    for gr, x, idx, step, res in graphs:
        for a, b in zip(res, step()):
            assert torch.equal(a, b)


def test_refusals():
    dev = "cuda"
    idx = torch.zeros((4, 2), dtype=torch.int32, device=dev)
    x = torch.zeros((4, 8), device=dev)
    y = torch.zeros((8, 8), device=dev)
    pos = torch.arange(8, dtype=torch.int32, device=dev)
    w = torch.ones((4, 2), device=dev)
    bad = [
        lambda: moe.permute(x, idx.long(), 4),                       # ids of another type
        lambda: moe.permute(x[:3], idx, 4),                          # rows do not match
        lambda: moe.permute(x.double(), idx, 4),
        lambda: moe.permute(x.t().contiguous().t(), idx, 4),         # strided rows
        lambda: moe.permute(x.cpu(), idx, 4),
        lambda: moe.permute(x, idx, 4, out=y.half()),
        lambda: moe.permute(x, idx, 4, out=y[:6]),
        lambda: moe.permute(x, idx, 0),
        lambda: moe.permute(x, idx, 1025),
        lambda: moe.permute(x, torch.zeros((4, 33), dtype=torch.int32, device=dev), 64),
        lambda: moe.permute_backward(y, pos[:7], 4, 2),
        lambda: moe.permute_backward(y, pos, 4, 2, out_dtype=torch.float64),
        lambda: moe.permute_backward(y[:, ::2], pos, 4, 2),
        lambda: moe.combine(y[:, ::2], pos, w, 4, 2),
        lambda: moe.combine(y, pos[:7], w, 4, 2),
        lambda: moe.combine(y, pos, w.half(), 4, 2),
        lambda: moe.combine(y, pos, w.cpu(), 4, 2),
        lambda: moe.combine(y, pos.cpu(), w, 4, 2),
        lambda: moe.combine(y, pos, w, 4, 2, y_shared=x.half()),
        lambda: moe.combine(y, pos, w, 4, 2, out_dtype=torch.float64),
        lambda: moe.combine_backward(x[:3], y, pos, w, 4, 2),
        lambda: moe.combine_backward(x, y, pos, w.double(), 4, 2),
        lambda: moe.combine_backward(x, y, pos, w, 4, 2, dy=y.half()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(_lib.VfmoeError) as e:
            call()
        assert e.value.code == _lib.ERR_INVALID, i
    torch.cuda.synchronize()


def test_outputs_that_overlap_inputs_are_refused():
    """One lane a token and square matrices make shapes that fit in place: the kernels would read rows others wrote."""
    T, H = 16, 64
    idx = torch.zeros((T, 1), dtype=torch.int32, device="cuda")
    buf = torch.zeros(T * H + 64, device="cuda")
    x, near = buf[:T * H].view(T, H), buf[64:].view(T, H)
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    y = torch.zeros((T, H), device="cuda")
    m = moe.q4_quantize(torch.randn(H, H, device="cuda"), group=32)
    bad = [
        lambda: moe.permute(x, idx, 4, out=x),
        lambda: moe.permute(x, idx, 4, out=near),
        lambda: moe.permute(near, idx, 4, out=x),
        lambda: moe.combine_backward(x, y, pos, None, T, 1, dy=x),
        lambda: moe.combine_backward(y, x, pos, None, T, 1, dy=near),
        lambda: moe.q4_matvec(x, m, out=x),
        lambda: moe.q4_matvec(near, m, out=x),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(_lib.VfmoeError, match="overlaps") as e:
            call()
        assert e.value.code == _lib.ERR_INVALID, i
    dy, _ = moe.combine_backward(y, x, pos, None, T, 1, dy=x)                 # the rows themselves are allowed
    assert dy.data_ptr() == x.data_ptr()
    halves = torch.zeros((2 * T, H), device="cuda")                            # neighbours in one buffer are apart
    moe.permute(halves[:T], idx, 4, out=halves[T:])
    moe.q4_matvec(halves[T:], m, out=halves[:T])
    torch.cuda.synchronize()
