"""4-bit matrices with group scales: quantize, dequantize and the products, against their definitions in 64 bits.

Bounds (v = 2^-24, S = sum |w| |x| of an output, u = finfo(dtype).eps / 2).  q - z and x are exact in the
kernel's operands.  A tensor-core step adds 16 products and the running sum, each possibly cut to 24 bits at the
largest one's exponent: 17 * 2v times the block's sum.  A block of 32 takes 2 steps (6 for fp32 x, which goes in three parts),
so its partial sum is off by at most 68 v (204 v) of its S; its scaling and the sum over K / 32 blocks add (K / 32 + 1) v,
the sum over warps fewer than 8 v.  Together below (K / 16 + 80) v S, and (K / 16 + 300) v S for fp32 x; a plain
loop over K / 32 values a lane stays below the same.  The store rounds once: u.
silu has slope at most 1.1: |d(silu(g) u)| <= 1.1 dg |u| + |silu(g)| du, and expf, the division and the products
another 8 v.
"""

import numpy as np
import pytest
import torch

from vybforge_b200 import _lib, moe

pytestmark = pytest.mark.gpu
V = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(lead, N, K, G, sdtype, zeros, g):
    q = torch.randint(0, 256, (*lead, N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = ((0.5 + torch.rand((*lead, K // G, N), generator=g, device="cuda")) * 0.01).to(sdtype)
    s[..., ::3] *= -1.0                                   # scales may be negative
    z = torch.randint(0, 16, (*lead, K // G, N), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return moe.Q4Matrix(q, s, z)


def dense64(m):
    """fp64 [.., N, K]."""
    q = torch.stack((m.codes & 15, m.codes >> 4), -1).flatten(-2).double()
    z = 8.0 if m.zeros is None else (m.zeros & 15).double().transpose(-1, -2).repeat_interleave(m.group, -1)
    return (q - z) * m.scales.double().transpose(-1, -2).repeat_interleave(m.group, -1)


def sum_err(K, dtype, S):
    return (K / 16 + (300 if dtype == torch.float32 else 80)) * V * S


def within(got, want, err, dtype):
    info = torch.finfo(dtype)
    tol = err + info.eps / 2 * (want.abs() + err) + info.smallest_normal * info.eps / 2
    d = (got.double() - want).abs()
    assert bool((d <= tol).all()), f"worst {float((d / tol).max()):.3g} of the bound"


def product64(w, x, dtype):
    """(exact, error bound) of x w^T, rows of x and w in fp64."""
    return x @ w.T, sum_err(x.shape[1], dtype, x.abs() @ w.abs().T)


def swiglu64(g, eg, u, eu, limit):
    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    a = g * torch.sigmoid(g)
    h = a * u
    return h, 1.1 * eg * (u.abs() + eu) + a.abs() * eu + 8 * V * h.abs()


SHAPES = [(16, 32, 32), (48, 96, 32), (64, 192, 64), (128, 384, 128), (80, 1056, 32), (272, 2176, 128), (1040, 320, 64),
          (16, 4096, 128), (4096, 64, 64)]


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 16, 17, 33, 64, 150])
@pytest.mark.parametrize("N,K,G", SHAPES)
def test_dense_product(N, K, G, n):
    for i, dtype in enumerate(DTYPES):
        g = gen(n + N + i)
        m = make((), N, K, G, (torch.float16, torch.bfloat16)[(n + i) % 2], (n + N // 16 + i) % 2 == 0, g)
        x = torch.randn(n, K, generator=g, device="cuda").to(dtype)
        want, err = product64(dense64(m), x.double(), dtype)
        for out in (dtype, torch.float32):
            y = moe.q4_matvec(x, m, out_dtype=out)
            within(y, want, err, out)
        assert torch.equal(y, moe.q4_matvec(x, m, out_dtype=torch.float32))      # the same bits every time


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,K,G", SHAPES)
def test_small_integers_are_exact(N, K, G, dtype, zeros):
    """Integer rows and scales of powers of two: every sum is exact, so every output is, whatever the order."""
    g = gen(1)
    m = make((), N, K, G, torch.bfloat16, zeros, g)
    m.scales.copy_(2.0 ** torch.randint(-3, 4, m.scales.shape, generator=g, device="cuda"))
    for n in (1, 5, 24):
        x = torch.randint(-4, 5, (n, K), generator=g, device="cuda").to(dtype)
        want = x.double() @ dense64(m).T                   # at most 4096 * 15 * 8 * 4 in steps of 1/8: 24 bits
        assert torch.equal(moe.q4_matvec(x, m, out_dtype=torch.float32).double(), want)


def expert_rows(E, T, k, mode, g):
    if mode == "one":
        idx = torch.full((T, k), E - 1, dtype=torch.int32, device="cuda")
    else:
        idx = torch.rand(T, E, generator=g, device="cuda").topk(k).indices.int()
        if mode == "dropped":
            idx[torch.rand(T, k, generator=g, device="cuda") < 0.4] = -1
        if mode == "none":
            idx[:] = -1
    return idx


@pytest.mark.parametrize("mode", ["plain", "dropped", "one", "none"])
@pytest.mark.parametrize("E,T,k,N,K,G", [(1, 5, 1, 32, 96, 32), (4, 1, 2, 64, 128, 128), (16, 40, 4, 48, 192, 64),
                                         (300, 9, 8, 32, 160, 32), (5, 150, 3, 96, 256, 128), (1024, 3, 16, 16, 64, 64)])
def test_experts(E, T, k, N, K, G, mode):
    for i, dtype in enumerate(DTYPES):
        g = gen(E + T + i)
        zeros, sd = (T + i) % 2 == 0, (torch.float16, torch.bfloat16)[i % 2]
        gate, up = make((E,), N, K, G, sd, zeros, g), make((E,), N, K, G, sd, zeros, g)
        x = torch.randn(T, K, generator=g, device="cuda").to(dtype)
        idx = expert_rows(E, T, k, mode, g)
        xs, plan = moe.permute(x, idx, E)
        off = plan.offsets.tolist()
        n = off[-1]
        wg, wu = dense64(gate), dense64(up)
        x64 = x.double()
        want, err, hw, he = (torch.zeros(T * k, N, dtype=torch.float64, device="cuda") for _ in range(4))
        limit = 0.2
        for e in range(E):
            r = slice(off[e], off[e + 1])
            if off[e] == off[e + 1]:
                continue
            rows = x64[plan.perm_tok[r].long()]
            want[r], err[r] = product64(wg[e], rows, dtype)
            u, eu = product64(wu[e], rows, dtype)
            hw[r], he[r] = swiglu64(want[r], err[r], u, eu, limit)
        fill = torch.full((T * k, N), 3.0, dtype=dtype, device="cuda")
        y = moe.q4_matvec(xs, gate, offsets=plan.offsets, out=fill.clone())
        within(y[:n], want[:n], err[:n], dtype)
        assert bool((y[n:] == 3.0).all())
        y2 = moe.q4_matvec(x, gate, offsets=plan.offsets, row_map=plan.perm_tok, out=fill.clone())
        assert torch.equal(y, y2)                          # the unsorted rows read in place
        h = moe.q4_matvec(x, gate, up=up, limit=limit, offsets=plan.offsets, row_map=plan.perm_tok, out=fill.clone(),
                          out_dtype=dtype)
        within(h[:n], hw[:n], he[:n], dtype)
        assert bool((h[n:] == 3.0).all())


# A dense call's layout goes by the channels (N = 208: warps along K, 8 of them; 4,752: one tile of channels, 4 warps along K;
# 9,488: two tiles, or with gate and up four; 18,960: four; a few more than 64, 128 and 512 in each) and by the rows (1: held in
# registers; 5: one tile of 8; 13: 16 rows, along K or from 9,472 channels on with x shared by warps; 45: 32 and 13 rows, the
# same), each for every type of x, group, type of scale, and with or without gate and up: these are all kernels there are.
# K is 19 chunks of 128 and a part of one, so every ring turns and ends inside a chunk.
@pytest.mark.parametrize("sdtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("N", [208, 4752, 9488, 18960])
def test_every_layout_of_a_dense_product(N, G, sdtype):
    K = 19 * 128 + {32: 96, 64: 64, 128: 0}[G]
    g = gen(N + G)
    for zeros in (False, True):
        gate, up = make((), N, K, G, sdtype, zeros, g), make((), N, K, G, sdtype, zeros, g)
        wg, wu = dense64(gate), dense64(up)
        for dtype in DTYPES:
            for n in (1, 5, 13, 45):
                x = torch.randn(n, K, generator=g, device="cuda").to(dtype)
                a, ea = product64(wg, x.double(), dtype)
                b, eb = product64(wu, x.double(), dtype)
                within(moe.q4_matvec(x, gate), a, ea, dtype)
                want, err = swiglu64(a, ea, b, eb, 2.0)
                within(moe.q4_matvec(x, gate, up=up, limit=2.0), want, err, dtype)


# The same for sorted rows, whose layout goes by the rows a matrix has on average: held, 8, 16 along K, 16 and 32 with shared x,
# 32 along K; and matrices with many times that ("one": all rows to one matrix, its tiles one after the other).
@pytest.mark.parametrize("mode", ["plain", "dropped", "one"])
@pytest.mark.parametrize("E,T,k,N,G", [(64, 2, 8, 624, 32), (64, 2, 8, 1200, 64), (64, 2, 8, 1200, 128), (16, 8, 4, 624, 128),
                                       (16, 8, 4, 1200, 32), (16, 8, 4, 1200, 64), (16, 24, 4, 80, 64), (16, 24, 4, 624, 32),
                                       (16, 24, 4, 640, 128), (16, 48, 4, 624, 64), (16, 48, 4, 1200, 32), (16, 48, 4, 1200, 128)])
def test_every_layout_of_sorted_rows(E, T, k, N, G, mode):
    K = 10 * 128 + {32: 96, 64: 64, 128: 0}[G]
    for i, dtype in enumerate(DTYPES):
        g = gen(E + T + N + i)
        zeros, sd = (G // 32 + i) % 2 == 0, (torch.bfloat16, torch.float16)[i % 2]
        gate, up = make((E,), N, K, G, sd, zeros, g), make((E,), N, K, G, sd, zeros, g)
        x = torch.randn(T, K, generator=g, device="cuda").to(dtype)
        _, plan = moe.permute(None, expert_rows(E, T, k, mode, g), E)
        off = plan.offsets.tolist()
        n = off[-1]
        y = moe.q4_matvec(x, gate, offsets=plan.offsets, row_map=plan.perm_tok, out=torch.full((T * k, N), 3.0, dtype=dtype,
                                                                                               device="cuda"))
        h = moe.q4_matvec(x, gate, up=up, limit=0.5, offsets=plan.offsets, row_map=plan.perm_tok)
        for e in range(E):
            r = slice(off[e], off[e + 1])
            if off[e] == off[e + 1]:
                continue
            rows = x[plan.perm_tok[r].long()].double()
            m = [moe.Q4Matrix(w.codes[e], w.scales[e], None if w.zeros is None else w.zeros[e]) for w in (gate, up)]
            a, ea = product64(dense64(m[0]), rows, dtype)
            b, eb = product64(dense64(m[1]), rows, dtype)
            within(y[r], a, ea, dtype)
            want, err = swiglu64(a, ea, b, eb, 0.5)
            within(h[r], want, err, dtype)
        assert bool((y[n:] == 3.0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("G", [32, 64, 128])
def test_rows_near_the_end_of_the_range(G, dtype):
    """Group sums are formed before the scale: they hold while 15 G max|x| stays within fp32, as documented."""
    g = gen(13)
    m = make((), 48, 512, G, torch.bfloat16, True, g)
    m.scales.copy_(2.0 ** -torch.randint(9, 12, m.scales.shape, generator=g, device="cuda"))
    x = (torch.rand(5, 512, generator=g, device="cuda") * 2 - 1) * (3.3e38 / (15 * G))
    x = x.to(dtype)
    want, err = product64(dense64(m), x.double(), dtype)
    within(moe.q4_matvec(x, m), want, err, dtype)


@pytest.mark.parametrize("n", [1, 12, 40])
def test_dense_gate_up(n):
    g = gen(n)
    for dtype in DTYPES:
        gate, up = (make((), 96, 512, 64, torch.float16, True, g) for _ in range(2))
        x = torch.randn(n, 512, generator=g, device="cuda").to(dtype) * 4
        a, ea = product64(dense64(gate), x.double(), dtype)
        b, eb = product64(dense64(up), x.double(), dtype)
        for limit in (10.0, 0.5, float("inf")):
            want, err = swiglu64(a, ea, b, eb, limit)
            within(moe.q4_matvec(x, gate, up=up, limit=limit), want, err, dtype)


def test_row_map_outside_reads_zeros():
    g = gen(3)
    m = make((), 32, 128, 64, torch.bfloat16, True, g)
    x = torch.randn(4, 128, generator=g, device="cuda")
    at = torch.tensor([2, -1, 0, 4, 2, 1 << 30], dtype=torch.int32, device="cuda")
    y = moe.q4_matvec(x, m, row_map=at)
    ref = moe.q4_matvec(x, m)
    for r, i in enumerate(at.tolist()):
        assert torch.equal(y[r], ref[i] if 0 <= i < 4 else torch.zeros_like(ref[0]))
    none = moe.q4_matvec(x[:0], m, row_map=torch.full((3,), -1, dtype=torch.int32, device="cuda"))
    assert none.shape == (3, 32) and bool((none == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nans_stay_in_their_row(dtype):
    """A row's infinity or NaN makes its own outputs so (codes that meet it are not zero) and no other's."""
    g = gen(4)
    m = make((), 64, 256, 32, torch.bfloat16, False, g)
    m.codes |= 0x99                                        # q >= 9: q - 8 > 0 everywhere
    m.scales.abs_()
    x = torch.randn(9, 256, generator=g, device="cuda").to(dtype)
    x2 = x.clone()
    x2[2, 77], x2[4, 200], x2[8, 0] = float("inf"), float("nan"), float("-inf")
    y, y2 = moe.q4_matvec(x, m), moe.q4_matvec(x2, m)
    assert bool((y2[2] == float("inf")).all()) and bool(y2[4].isnan().all()) and bool((y2[8] == float("-inf")).all())
    for r in (0, 1, 3, 5, 6, 7):
        assert torch.equal(y[r], y2[r])


@pytest.mark.parametrize("limit", [10.0, float("inf")])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [64, 9504])                  # one tile a warp, and four
@pytest.mark.parametrize("n", [2, 9, 40])
def test_gate_up_keeps_nans_and_infinities(n, N, dtype, limit):
    """The clamps of the fused SwiGLU pass a NaN on (max and min that drop it would store numbers that look sound), as
    its definition does; a row of +inf gives the clamped product, one of -inf silu(-inf) = -inf / inf = NaN."""
    g = gen(11)
    gate, up = (make((), N, 672, 32, torch.bfloat16, False, g) for _ in range(2))
    for m in (gate, up):
        m.codes |= 0x99                                    # q - 8 > 0 everywhere
        m.scales.abs_()
    blind = moe.Q4Matrix(torch.full_like(up.codes, 0x88), up.scales)   # q - 8 = 0: 0 for finite rows, NaN for infinite
    x = torch.randn(n, 672, generator=g, device="cuda").to(dtype)
    bad = {0: float("nan"), 1: float("inf")}
    if n > 2:
        bad[8] = float("-inf")
    x2 = x.clone()
    for r, v in bad.items():
        x2[r, 77 * (r + 1) % 672] = v
    clean, got = moe.q4_matvec(x, gate, up=up, limit=limit), moe.q4_matvec(x2, gate, up=up, limit=limit)
    assert bool(got[0].isnan().all())
    if limit == float("inf"):
        assert bool((got[1] == limit).all())
    else:                                                  # silu(10) * 10: the formula's error as in swiglu64, rounded once
        want = torch.full((N,), limit * limit / (1.0 + np.exp(-limit)), dtype=torch.float64, device="cuda")
        within(got[1], want, 8 * V * want, dtype)
    if n > 2:
        assert bool(got[8].isnan().all())
    for r in range(n):
        if r not in bad:
            assert torch.equal(got[r], clean[r]) and bool(got[r].isfinite().all())
    half = moe.q4_matvec(x2, gate, up=blind, limit=limit)  # a NaN of the up product alone
    for r in range(n):
        assert bool(half[r].isnan().all()) if r in bad else bool((half[r] == 0).all())


def test_fp32_rows_keep_their_bits():
    """fp32 rows that differ from bf16 ones in their last bits: the product follows them."""
    g = gen(5)
    m = make((), 32, 2048, 128, torch.bfloat16, True, g)
    x = torch.randn(3, 2048, generator=g, device="cuda")
    d = (x - x.bfloat16().float())
    want = d.double() @ dense64(m).T
    got = moe.q4_matvec(x, m).double() - moe.q4_matvec(x.bfloat16().float(), m).double()
    S = x.double().abs() @ dense64(m).abs().T
    assert bool(((got - want).abs() <= 2 * sum_err(2048, torch.float32, S) + 4 * V * S).all())


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("G", [32, 64, 128])
def test_quantize_and_dequantize(G, zeros):
    for src in DTYPES:
        for sd in (torch.float16, torch.bfloat16):
            g = gen(G)
            w = (torch.randn(2, 48, 256, generator=g, device="cuda") * 0.05).to(src)
            w[0, 3] = 0.0                                  # a row of zeros
            w[1, 5] = w[1, 5].abs() + 0.01                 # a one-sided row
            m = moe.q4_quantize(w, group=G, scale_dtype=sd, zeros=zeros)
            d = moe.q4_dequant(m)
            assert torch.equal(d.double(), dense64(m))     # an 11-bit scale times 5 bits: exact in fp32
            for out in (torch.float16, torch.bfloat16):
                assert torch.equal(moe.q4_dequant(m, out), d.to(out))
            assert bool((d[0, 3] == 0).all())
            # half a step of the code, or of the zero point, and what the 16-bit scale lost at the range's end
            s = m.scales.float().transpose(-1, -2).repeat_interleave(G, -1)
            u = torch.finfo(sd).eps / 2
            reach = 15.0 if zeros else 7.0
            step = s.abs() * ((1.0 if zeros else 0.5) + 2 * reach * u + 16 * V) + 1e-7
            assert bool(((d - w.float()).abs() <= step).all())
            if zeros:
                assert int(m.zeros.max()) <= 15


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("sd", [torch.float16, torch.bfloat16])
def test_quantize_the_largest_finite_weights(sd, zeros):
    """Finite weights give finite codes and scales: a scale past fp16's range takes its largest value and the far elements
    the end of the code range, and a range that passes fp32 itself is no infinite scale."""
    G, N, K = 64, 32, 256
    g = gen(12)
    w = torch.randn(N, K, generator=g, device="cuda")
    w[:16] *= 1e6                                          # scales of about 2e5 to 4e5 where fp16 ends at 65,504
    w[16:] = torch.where(w[16:] < 0, -2.5e38, 2.5e38) * torch.rand(16, K, generator=g, device="cuda")
    w[:, ::G], w[:, 1::G] = w[:, ::G].abs(), -w[:, 1::G].abs()   # both signs in every group
    m = moe.q4_quantize(w, group=G, scale_dtype=sd, zeros=zeros)
    d = moe.q4_dequant(m)
    assert bool(m.scales.isfinite().all()) and bool(d.isfinite().all())
    s = m.scales.double().transpose(-1, -2).repeat_interleave(G, -1)
    z = 8.0 if m.zeros is None else m.zeros.double().transpose(-1, -2).repeat_interleave(G, -1)
    reach = (w.double().clamp(-z * s, (15.0 - z) * s) - d.double()).abs()      # half a step, and the quotient's rounding
    assert bool((reach <= s * (0.5 + 16 * V)).all())
    if sd == torch.float16:
        assert bool((m.scales == 65504).all())
    else:                                                  # as in test_quantize_and_dequantize
        u, top = torch.finfo(sd).eps / 2, 15.0 if zeros else 7.0
        step = s * ((1.0 if zeros else 0.5) + 2 * top * u + 16 * V)
        assert bool(((d - w).double().abs() <= step).all())


def test_no_rows_and_one_stream():
    g = gen(6)
    m = make((), 32, 64, 32, torch.bfloat16, False, g)
    assert moe.q4_matvec(torch.empty((0, 64), device="cuda"), m).shape == (0, 32)
    x = torch.randn(5, 64, generator=g, device="cuda")
    ref = moe.q4_matvec(x, m)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = moe.q4_matvec(x, m)
    side.synchronize()
    assert torch.equal(y, ref)


def test_offsets_beyond_32_bits():
    """A stack of 2.4 GB of codes: the last matrices lie past 2^31 bytes, their elements past 2^32."""
    E, N, K, G = 200, 4096, 6144, 128
    g = gen(7)
    m = make((E,), N, K, G, torch.bfloat16, True, g)
    idx = torch.tensor([[0, 150, 199], [199, 198, 3]], dtype=torch.int32, device="cuda")
    x = torch.randn(2, K, generator=g, device="cuda", dtype=torch.bfloat16)
    _, plan = moe.permute(None, idx, E)
    y = moe.q4_matvec(x, m, offsets=plan.offsets, row_map=plan.perm_tok, out_dtype=torch.float32)
    ids = idx.reshape(-1).long()
    for lane in range(6):
        e = int(ids[lane])
        one = moe.Q4Matrix(m.codes[e], m.scales[e], m.zeros[e])
        want, err = product64(dense64(one), x[lane // 3:lane // 3 + 1].double(), torch.bfloat16)
        within(y[int(plan.pos_of[lane])], want[0], err[0], torch.float32)


@pytest.mark.parametrize("dtype,T", [(torch.bfloat16, 1), (torch.bfloat16, 70), (torch.float32, 6)])
def test_a_token_through_its_experts_and_back(dtype, T):
    """permute -> gate/up + SwiGLU -> down -> combine, as a decode step runs them, captured once and replayed
    on other rows and ids; every stage against its definition on its own input."""
    E, k, H, I, G = 24, 4, 256, 128, 64
    g = gen(8)
    gate, up = make((E,), I, H, G, torch.float16, True, g), make((E,), I, H, G, torch.float16, True, g)
    down = make((E,), H, I, G, torch.float16, True, g)
    x = torch.zeros(T, H, device="cuda", dtype=dtype)
    idx = torch.zeros(T, k, device="cuda", dtype=torch.int32)
    w = torch.zeros(T, k, device="cuda")

    def step():
        _, plan = moe.permute(None, idx, E)
        h = moe.q4_matvec(x, gate, up=up, offsets=plan.offsets, row_map=plan.perm_tok)
        y = moe.q4_matvec(h, down, offsets=plan.offsets, out_dtype=torch.float32)
        return plan, h, y, moe.combine(y, plan.pos_of, w, T, k, out_dtype=torch.float32)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            plan, h, y, out = step()
    torch.cuda.synchronize()
    for seed in (1, 2):
        gs = gen(seed)
        x.copy_(torch.randn(T, H, generator=gs, device="cuda"))
        idx.copy_(expert_rows(E, T, k, "dropped" if seed == 2 else "plain", gs))
        w.copy_(torch.rand(T, k, generator=gs, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        n = int(plan.offsets[-1])
        e = torch.searchsorted(plan.offsets[1:].contiguous(), torch.arange(n, dtype=torch.int32, device="cuda"), right=True)
        mats = [dense64(m) for m in (gate, up, down)]
        tok = plan.perm_tok[:n].long()
        final = torch.zeros(T, H, dtype=torch.float64, device="cuda")
        for r in range(n):
            xr, hr = x[tok[r]].double().view(1, -1), h[r].double().view(1, -1)
            a, ea = product64(mats[0][e[r]], xr, dtype)
            b, eb = product64(mats[1][e[r]], xr, dtype)
            hw, he = swiglu64(a, ea, b, eb, 10.0)
            within(h[r], hw[0], he[0], dtype)
            yw, ye = product64(mats[2][e[r]], hr, dtype)
            within(y[r], yw[0], ye[0], torch.float32)
        kept = (plan.pos_of >= 0).view(T, k)
        terms = torch.where(kept.unsqueeze(-1), w.double().unsqueeze(-1) *
                            y.double()[plan.pos_of.clamp(min=0).long()].view(T, k, H), 0.0)
        within(out, terms.sum(1), (k + 2) * V * terms.abs().sum(1), torch.float32)


def test_refusals():
    g = gen(9)
    m = make((), 32, 128, 32, torch.bfloat16, True, g)
    st = make((3,), 32, 128, 32, torch.bfloat16, True, g)
    x = torch.zeros(4, 128, device="cuda")
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    c, s, z = m.codes, m.scales, m.zeros
    odd = torch.empty(33, 128, device="cuda").view(-1)[1:4 * 128 + 1].view(4, 128)
    bad = [
        lambda: moe.q4_matvec(x[:, :64].contiguous(), m),
        lambda: moe.q4_matvec(x.t().contiguous().t(), m),
        lambda: moe.q4_matvec(x.double(), m),
        lambda: moe.q4_matvec(x.cpu(), m),
        lambda: moe.q4_matvec(odd, m),                                   # not 16-byte aligned
        lambda: moe.q4_matvec(x, m, out_dtype=torch.float64),
        lambda: moe.q4_matvec(x, m, out=torch.zeros(4, 16, device="cuda")),
        lambda: moe.q4_matvec(x, st),                                    # a stack without offsets
        lambda: moe.q4_matvec(x, st, offsets=off[:3]),
        lambda: moe.q4_matvec(x, st, offsets=off.long()),
        lambda: moe.q4_matvec(x, m, row_map=off.long()),
        lambda: moe.q4_matvec(x, m, up=moe.Q4Matrix(c, s)),              # other kind of zero points
        lambda: moe.q4_matvec(x, m, up=moe.Q4Matrix(c, s.half(), z)),    # other scale type
        lambda: moe.q4_matvec(x, m, up=m, limit=0.0),
        lambda: moe.q4_matvec(x, m, up=m, limit=float("nan")),
        lambda: moe.Q4Matrix(c.int(), s, z),
        lambda: moe.Q4Matrix(c, s.float(), z),
        lambda: moe.Q4Matrix(c, s[:, :16], z),
        lambda: moe.Q4Matrix(c, s[:3].contiguous(), z[:3].contiguous()),
        lambda: moe.Q4Matrix(c, s, z.to(torch.int8)),
        lambda: moe.q4_matvec(x, moe.Q4Matrix(c[:24].contiguous(), s[:, :24].contiguous())),   # N % 16
        lambda: moe.q4_matvec(x, moe.Q4Matrix(c, s[:2].contiguous()[:, :].repeat_interleave(4, 0))),   # groups of 16
        lambda: moe.q4_quantize(x, group=48),
        lambda: moe.q4_quantize(x.long()),
        lambda: moe.q4_dequant(m, torch.float64),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(_lib.VfmoeError) as err:
            call()
        assert err.value.code == _lib.ERR_INVALID, i
    torch.cuda.synchronize()
