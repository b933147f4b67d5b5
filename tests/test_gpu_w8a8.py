"""-m gpu: the W8A8 operators (ds_gemm_i8, ds_rmsnorm_rows, ds_quantize_rows_i8, ds_dequantize_rows_i8) against the definitions in 64 bits.

Tolerances.  H(t) = half a step of a rounding to t (relative): fp16 2^-11, fp32 2^-24; a subnormal fp16 result is off by at most 2^-25.
  product   p = acc * a_scale * w_scale: the integer sum is exact, its conversion and the two products round (3 H32 |p|), the bias adds one
            rounding of the result (H32 (|p| + |b|)), the residual one more: 5 H32 (|p| + |b| + |r|) in all, then H(out) |out|.
            SiLU: slope <= 1.1, and x / (1 + e^-x) itself: exp 2 ulp (4 H32), sum, quotient: 8 H32 |silu|; with an fp16 result e^-x is
            2^(-1.4427 x), whose argument rounds twice (constant and product): 2 H32 |x| |silu| more.  GEGLU: value * gelu(gate): the
            errors of value and gate (slope <= 1.13) are carried, 1 + erf is off by at most 8 H32 absolute, hence gelu by 4 H32 |gate|, and
            three products: 4 H32 |result|.  With an fp16 result gelu comes from a fit of erfc that is within 1.6e-5 of it (found on 200 000 points,
            8.6e-6 ln 2 by the fit and its 32-bit evaluation), the 2^-q within 2e-5: 2e-5 |gate| / 2 erfc(|gate| / sqrt 2) more.
  8 bits    q has to be EQUAL: the kernel rounds the exact quotient.  scale: one rounding of a 64-bit value, H32, doubled for slack in sums.
  norm y    h, root, gamma: at most five fp32 roundings (5 H32) before H(out).
  sum       H32 + H(out).
"""
import contextlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

H16, H32 = 2.0 ** -11, 2.0 ** -24
SUB = {torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}
HALF = {torch.float16: H16, torch.float32: H32}
F16, F32 = torch.float16, torch.float32


def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    return torch.device("cuda:0")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(shape, seed):
    return torch.randint(-128, 128, shape, generator=gen(seed), dtype=torch.int16).to(torch.int8)


def normal(shape, seed, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=gen(seed)) * scale).to(dtype)


def product_ref(a, w, sa, sw, bias, residual, act, out=F16):
    """(result, tolerance before the output's rounding) in 64 bits."""
    p = (a.double() @ w.double().t()) * sa.double()[:, None] * sw.double()
    b = torch.zeros_like(p) if bias is None else bias.double().expand_as(p)
    v, e = p + b, 5 * H32 * (p.abs() + b.abs())
    if act == "silu":
        s = v * torch.sigmoid(v)
        e = 1.1 * e + 8 * H32 * s.abs() + (2 * H32 * v.abs() * s.abs() if out == F16 else 0.0)
        v = s
    elif act == "geglu":
        m, n = v.shape
        vv, ee = v.view(m, n // 64, 2, 32), e.view(m, n // 64, 2, 32)
        x, g, ex, eg = vv[:, :, 0], vv[:, :, 1], ee[:, :, 0], ee[:, :, 1]
        gelu = 0.5 * g * torch.erfc(-g / math.sqrt(2.0))
        v = (x * gelu).reshape(m, n // 2)
        fit = 2e-5 * g.abs() / 2 * torch.erfc(g.abs() / math.sqrt(2.0)) if out == F16 else 0.0
        e = (ex * gelu.abs() + x.abs() * (1.13 * eg + 4 * H32 * g.abs() + fit) + ex * 1.13 * eg).reshape(m, n // 2) + 4 * H32 * v.abs()
    if residual is not None:
        r = residual.double()
        v, e = v + r, e + 2 * H32 * (v.abs() + r.abs())
    return v, e


def close(got, ref, before, dtype):
    assert got.dtype == dtype and tuple(got.shape) == tuple(ref.shape)
    tol = (before + HALF[dtype] * (ref.abs() + before) + SUB[dtype])
    off = (got.double().cpu() - ref).abs()
    worst = float((off / tol).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{worst} of the tolerance at {int((off / tol).argmax())}"


def product_case(m, n, k, seed, bias=True, residual=None, act="none"):
    cols = n // 2 if act == "geglu" else n
    a, w = ints((m, k), seed), ints((n, k), seed + 1)
    sa, sw = torch.rand(m, generator=gen(seed + 2)) * 0.02 + 1e-3, torch.rand(n, generator=gen(seed + 3)) * 0.02 / math.sqrt(max(k, 1)) + 1e-4
    b = normal((n,), seed + 4) if bias else None
    r = normal((m, cols), seed + 5, residual) if residual is not None else None
    return a, w, sa, sw, b, r


EPI = {"none": 0, "silu": 2, "geglu": 1}


def run_product(c, act="none", out_dtype=F16, **kw):
    from dynamicscaler_amd import ops
    d = dev()
    a, w, sa, sw, b, r = [None if t is None else t.to(d) for t in c]
    return ops.gemm_i8(a, w, sa, sw, bias=b, residual=r, epilogue=EPI[act], out_dtype=out_dtype, **kw)


# one row, few rows, whole tiles and one more than them, inner axes below / at / above a chunk (16), a slice (64) and a step (128) of k
SIZES = [(1, 1, 1), (1, 5, 16), (2, 64, 15), (3, 64, 127), (16, 16, 64), (17, 33, 129), (1, 1280, 1280), (16, 320, 5120), (31, 100, 320),
         (77, 512, 1024), (64, 257, 33), (65, 130, 48), (127, 64, 128), (129, 65, 257), (128, 128, 256), (255, 320, 320), (257, 256, 384),
         (300, 641, 1273), (512, 512, 640), (640, 1280, 144), (1000, 96, 2560), (2049, 320, 320)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("out_dtype,residual", [(F16, None), (F16, F16), (F32, F32), (F32, F16), (F16, F32)])
def test_product(m, n, k, out_dtype, residual):
    c = product_case(m, n, k, m + n + k, residual=residual)
    got = run_product(c, out_dtype=out_dtype)
    close(got, *product_ref(*c, "none"), out_dtype)


@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (5, 128, 100), (16, 2560, 320), (77, 640, 1024), (130, 192, 96), (257, 5120, 320), (600, 1024, 640), (2050, 640, 320)])
@pytest.mark.parametrize("act", ["silu", "geglu"])
@pytest.mark.parametrize("out_dtype", [F16, F32])
@pytest.mark.parametrize("bias", [True, False])
def test_product_activations(m, n, k, act, out_dtype, bias):
    c = product_case(m, n, k, 7 * m + n + k, bias=bias, act=act)
    got = run_product(c, act=act, out_dtype=out_dtype)
    close(got, *product_ref(*c, act, out_dtype), out_dtype)


@pytest.mark.parametrize("m,k", [(2, 64), (40, 100), (300, 64), (300, 37), (2500, 64)])
def test_geglu_of_far_gates(m, k):
    """fp32 GEGLU relative to itself for gates down to where erfc leaves fp32: operands whose sums are one and whose scales are the values and gates,
    so that both are exact.  E = erfc(|gate| / sqrt 2) is off by at most 12 H32 E (8 in the formula's own roundings, 4 for the hardware's reciprocal and
    power of two), value * gate / 2 * (E or 2 - E) rounds four times, the result once."""
    from dynamicscaler_amd import ops
    d = dev()
    groups = 64
    gates = torch.cat([torch.linspace(-12.9, 12.9, 32 * groups - 32), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e-6, -1e-6, -5.5, -6.0] * 4)])
    gates = gates[torch.randperm(32 * groups, generator=gen(1))].view(groups, 32)
    values = (0.5 + 1.5 * torch.rand((groups, 32), generator=gen(2)))
    values[::3] *= 1e6
    a, w = torch.zeros((m, k), dtype=torch.int8), torch.zeros((64 * groups, k), dtype=torch.int8)
    a[:, k - 1] = 1
    w[:, k - 1] = 1
    sw = torch.stack([values, gates], dim=1).reshape(-1)
    got = ops.gemm_i8(a.to(d), w.to(d), torch.ones(m, device=d), sw.to(d), out_dtype=F32, epilogue=EPI["geglu"]).cpu()
    g = gates.double()
    ref = (values.double() * g / 2 * torch.erfc(-g / math.sqrt(2.0))).reshape(1, -1).expand(m, -1)
    e = torch.erfc(g.abs() / math.sqrt(2.0))
    factor = torch.where(g < 0, e, 2 - e)
    before = (12 * e / factor + 4).reshape(1, -1) * H32 * ref.abs()
    close(got, ref, before, F32)


@pytest.mark.parametrize("m,n,k", [(4, 40, 131071), (130, 70, 131071), (260, 256, 131056)])
def test_product_longest_sums_are_exact(m, n, k):
    """Every term 2^14: the sums reach 2^31 - 2^14 and have to come out whole (fp32 out, scales of one)."""
    d = dev()
    from dynamicscaler_amd import ops
    a = torch.full((m, k), -128, dtype=torch.int8, device=d)
    w = torch.full((n, k), -128, dtype=torch.int8, device=d)
    w[1::2] = 127
    one_m, one_n = torch.ones(m, device=d), torch.ones(n, device=d)
    got = ops.gemm_i8(a, w, one_m, one_n, out_dtype=F32)
    ref = torch.full((m, n), float(k * 128 * 128))
    ref[:, 1::2] = float(-k * 128 * 127)
    assert torch.equal(got.cpu(), ref)


@pytest.mark.parametrize("m,n,k,offs", [(33, 50, 70, (1, 3, 1, 1)), (300, 320, 320, (16, 32, 8, 8)), (300, 320, 320, (5, 0, 3, 1)), (9, 256, 512, (16, 16, 8, 4)),
                                        (257, 300, 128, (0, 7, 0, 5)), (2100, 256, 256, (16, 16, 4, 8))])
@pytest.mark.parametrize("out_dtype", [F16, F32])
def test_product_strides_and_neighbours(m, n, k, offs, out_dtype):
    """Operands and results as column slices of wider matrices, at aligned and unaligned offsets; what lies around the result stays."""
    from dynamicscaler_amd import ops
    d = dev()
    a, w, sa, sw, b, r = product_case(m, n, k, 11, residual=out_dtype)
    oa, ow, oc, orr = offs

    def inside(t, off, fill):
        wide = torch.full((t.shape[0] + 2, t.shape[1] + 2 * off + 7), fill, dtype=t.dtype, device=d)
        wide[1:-1, off:off + t.shape[1]] = t.to(d)
        return wide, wide[1:-1, off:off + t.shape[1]]

    A, W = inside(a, oa, 77)[1], inside(w, ow, -99)[1]
    R = inside(r, orr, 1e4)[1]
    wide, out = inside(torch.zeros(m, n, dtype=out_dtype), oc, 1234.0)
    got = ops.gemm_i8(A, W, sa.to(d), sw.to(d), bias=b.to(d), residual=R, out=out)
    assert got is out
    close(out, *product_ref(a, w, sa, sw, b, r, "none"), out_dtype)
    out.fill_(1234.0)
    assert bool((wide == 1234.0).all())


@pytest.mark.parametrize("m,n,k", [(3, 64, 64), (100, 320, 640), (1025, 320, 320)])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_product_in_place_residual(m, n, k, dtype):
    c = product_case(m, n, k, 5, residual=dtype)
    d = dev()
    stream = c[5].to(d)
    from dynamicscaler_amd import ops
    ops.gemm_i8(c[0].to(d), c[1].to(d), c[2].to(d), c[3].to(d), bias=c[4].to(d), residual=stream, out=stream)
    close(stream, *product_ref(*c, "none"), dtype)


@pytest.mark.parametrize("m,n,k", [(0, 16, 16), (4, 0, 16), (0, 0, 0)])
def test_product_of_nothing(m, n, k):
    c = product_case(m, n, k, 1)
    assert tuple(run_product(c).shape) == (m, n)


def test_product_without_an_inner_axis_is_the_bias():
    c = product_case(5, 64, 0, 1, residual=F16)
    got = run_product(c, out_dtype=F32)
    close(got, *product_ref(*c, "none"), F32)


@pytest.mark.parametrize("m,n,k", [(4, 48, 100), (200, 320, 320), (600, 512, 512)])
def test_product_rows_that_stand_for_zero_or_nan(m, n, k):
    """A scale of zero gives bias + residual, a NaN scale a row / column of NaN, and no other row or column notices."""
    a, w, sa, sw, b, r = product_case(m, n, k, 3, residual=F32)
    sa[1], sa[2], sw[3] = 0.0, float("nan"), float("inf")
    got = run_product((a, w, sa, sw, b, r), out_dtype=F32).cpu()
    assert bool(got[2].isnan().all())
    keep_m, keep_n = [i for i in range(m) if i != 2], [j for j in range(n) if j != 3]
    ref, e = product_ref(a[keep_m], w[keep_n], sa[keep_m], sw[keep_n], b[keep_n], r[keep_m][:, keep_n], "none")
    close(got[keep_m][:, keep_n], ref, e, F32)
    assert not bool(got[keep_m, 3].isfinite()[0]) or bool((a[0].int() * w[3].int()).sum() == 0)


def large_case(m, n, k, out_dtype, residual, act, seed=0):
    """Operands on the device, and the definition in 64 bits there (elementary operations; the integer sums are exact in float64)."""
    d = dev()
    g = torch.Generator(device=d).manual_seed(seed)
    a = torch.randint(-128, 128, (m, k), generator=g, device=d, dtype=torch.int16).to(torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, device=d, dtype=torch.int16).to(torch.int8)
    cols = n // 2 if act == "geglu" else n
    sa, sw = torch.rand(m, generator=g, device=d) * 0.02 + 1e-3, torch.rand(n, generator=g, device=d) * 0.02 / math.sqrt(k) + 1e-4
    b = torch.randn(n, generator=g, device=d)
    r = torch.randn((m, cols), generator=g, device=d).to(residual) if residual is not None else None
    return (a, w, sa, sw, b, r), product_ref(a, w, sa, sw, b, r, act, out_dtype)


# one size for each tile of the many-rows kernel (256 x 256, 128 x 128, 256 x 64, 128 x 64, 64 x 64; 128 x 128 and 64 x 64 through registers), with
# rows and columns that end inside a tile, the last K-step cut, results below and above the size from which they pass the cache by, a few rows
# against so many columns that the tiles have them
@pytest.mark.parametrize("m,n,k", [(8200, 1296, 1040), (16500, 2576, 144), (8200, 2576, 1296), (20500, 656, 336), (40970, 320, 320), (4100, 1296, 1296), (1030, 656, 656),
                                   (8211, 1297, 1043), (33000, 656, 333), (1030, 657, 655), (33, 20480, 656), (50, 4161, 4095)])
@pytest.mark.parametrize("out_dtype,residual,act", [(F16, None, "none"), (F16, F16, "none"), (F32, F32, "none"), (F32, None, "silu"), (F16, F32, "none"), (F16, None, "geglu"),
                                                    (F32, None, "geglu")])
def test_product_every_tile(m, n, k, out_dtype, residual, act):
    from dynamicscaler_amd import ops
    if act == "geglu":
        n = n // 64 * 64
    (a, w, sa, sw, b, r), (ref, before) = large_case(m, n, k, out_dtype, residual, act)
    got = ops.gemm_i8(a, w, sa, sw, bias=b, residual=r, epilogue=EPI[act], out_dtype=out_dtype)
    off = (got.double() - ref).abs()
    tol = before + HALF[out_dtype] * (ref.abs() + before) + SUB[out_dtype]
    assert got.dtype == out_dtype and float((off / tol).max()) <= 1.0
    if residual == out_dtype:                    # the residual stream in place
        assert ops.gemm_i8(a, w, sa, sw, bias=b, residual=r, epilogue=EPI[act], out=r) is r
        assert torch.equal(r, got)


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 31, 33, 48, 49, 64, 65])
@pytest.mark.parametrize("n,k", [(48, 64), (1280, 1280), (321, 1023), (130, 4095), (64, 13), (700, 66)])
@pytest.mark.parametrize("act", ["none", "geglu"])
def test_product_few_rows(m, n, k, act):
    """Rows around the few-rows kernel's groups of 16, K split over its waves unevenly, odd addresses, columns that end inside a group."""
    if act == "geglu":
        n = max(64, n // 64 * 64)
    c = product_case(m, n, k, m + n, residual=F16 if act == "none" else None, act=act)
    close(run_product(c, act=act), *product_ref(*c, act), F16)


@pytest.mark.parametrize("m,n,k", [(2057, 997, 1273), (2057, 1000, 1284), (1500, 1056, 4095)])
def test_product_with_and_without_copied_operands(m, n, k):
    """Odd rows laid out anew in the workspace (the usual call) or read as they lie (a call that names its stream has none): the same bits."""
    (a, w, sa, sw, b, r), (ref, before) = large_case(m, n, k, F32, F32, "none")
    from dynamicscaler_amd import ops
    got = ops.gemm_i8(a, w, sa, sw, bias=b, residual=r, out_dtype=F32)
    assert float(((got.double() - ref).abs() / (before + H32 * (ref.abs() + before))).max()) <= 1.0
    assert torch.equal(got, ops.gemm_i8(a, w, sa, sw, bias=b, residual=r, out_dtype=F32, stream=torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("act", ["none", "silu", "geglu"])
@pytest.mark.parametrize("out_dtype", [F16, F32])
def test_product_is_the_same_for_any_rows_of_the_launch(act, out_dtype):
    """Row m of a large launch equals the launch of row m alone, bit for bit (every kernel adds the same exact sum and ends with the same steps)."""
    a, w, sa, sw, b, _ = product_case(700, 384, 640, 9, act=act)
    whole = run_product((a, w, sa, sw, b, None), act=act, out_dtype=out_dtype)
    for lo, hi in ((0, 1), (3, 19), (100, 165), (0, 300), (699, 700)):
        assert torch.equal(whole[lo:hi], run_product((a[lo:hi], w, sa[lo:hi], sw, b, None), act=act, out_dtype=out_dtype))


@pytest.mark.parametrize("which", ["A", "out"])
def test_product_offsets_beyond_32_bits(which):
    """Rows that start beyond 2^31 elements of their tensor."""
    from dynamicscaler_amd import ops
    d = dev()
    c = product_case(3, 64, 128, 21)
    a, w, sa, sw, b, _ = [None if t is None else t.to(d) for t in c]
    ld = (1 << 30) + 64 + 3
    out = None
    if which == "A":
        big = torch.empty((3 * ld,), dtype=torch.int8, device=d)
        A = big.as_strided((3, 128), (ld, 1))
        A.copy_(a)
        a = A
    else:
        big = torch.empty((3 * ld,), dtype=F16, device=d)
        out = big.as_strided((3, 64), (ld, 1))
    close(ops.gemm_i8(a, w, sa, sw, bias=b, out=out), *product_ref(*c, "none"), F16)


# ------------------------------------------------------------------------------------------------ rows
def rows_ref(x, r, g, eps, norm):
    h = x.double() if r is None else x.double() + r.double()
    root = 1.0 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + eps) if norm else torch.ones(h.shape[0], 1, dtype=torch.float64)
    return h, (h * g.double() if norm else h), root


def eight_bits(t, root):
    top = t.abs().amax(dim=1, keepdim=True)
    q = torch.where(top > 0, torch.round(127.0 * t / torch.where(top > 0, top, torch.ones_like(top))), torch.zeros_like(t))
    return q, (top * root / 127.0)[:, 0]


def check_rows_i8(q, scale, t, root):
    rq, rs = eight_bits(t, root)
    assert q.dtype == torch.int8 and torch.equal(q.cpu().double(), rq)
    assert bool(((scale.cpu().double() - rs).abs() <= 2 * H32 * rs + 2.0 ** -149).all())


ROW_SIZES = [(1, 1), (2, 3), (1, 8), (3, 63), (5, 64), (7, 65), (4, 127), (9, 320), (3, 511), (33, 640), (1, 1280), (6, 1283), (2, 2047), (3, 2560),
             (2, 4099), (5, 5120), (1, 8192), (2, 8200), (2, 10240), (1, 16384), (2, 20011), (1, 40000)]


def row_inputs(m, n, seed, dtype):
    x = torch.randn((m, n), generator=gen(seed)) * torch.exp(torch.randn((n,), generator=gen(seed + 1)) * 0.7)
    return x.to(dtype)


@pytest.mark.parametrize("m,n", ROW_SIZES)
@pytest.mark.parametrize("xt,rt", [(F16, None), (F16, F16), (F16, F32), (F32, F32), (F32, F16), (F32, None)])
def test_norm(m, n, xt, rt):
    from dynamicscaler_amd import ops
    d = dev()
    x, g = row_inputs(m, n, m + n, xt), 1.0 + 0.2 * normal((n,), n)
    r = None if rt is None else normal((m, n), m, rt, 2.0)
    h, t, root = rows_ref(x, r, g, 1e-6, True)
    rd = None if r is None else r.to(d)
    q, scale, back = ops.rmsnorm_i8(x.to(d), g.to(d), eps=1e-6, residual=rd)
    check_rows_i8(q, scale, t, root)
    sums = [back]
    for ot in (F16, F32):
        y, back = ops.rmsnorm(x.to(d), g.to(d), eps=1e-6, residual=rd, out_dtype=ot)
        close(y, t * root, 5 * H32 * (t * root).abs(), ot)
        sums.append(back)
    for back in sums:
        if rt is None:
            assert back is None
        else:
            close(back, h, H32 * h.abs(), rt)


@pytest.mark.parametrize("m,n", ROW_SIZES)
@pytest.mark.parametrize("xt", [F16, F32])
def test_quantize_and_back(m, n, xt):
    from dynamicscaler_amd import ops
    d = dev()
    x = row_inputs(m, n, 2 * m + n, xt)
    q, scale = ops.quantize_rows_i8(x.to(d))
    check_rows_i8(q, scale, x.double(), torch.ones(m, 1, dtype=torch.float64))
    for ot in (F16, F32):
        y = ops.dequantize_rows_i8(q, scale, dtype=ot)
        v = q.cpu().double() * scale.cpu().double()[:, None]
        close(y, v, H32 * v.abs(), ot)
    assert bool(((y.double().cpu() - x.double()).abs() <= scale.cpu().double()[:, None] * (0.5 + 1e-4)).all())


def once(v):
    """fp64 to fp16 in one rounding (torch goes by way of fp32)."""
    import numpy as np
    with np.errstate(over="ignore"):
        return torch.from_numpy(v.numpy().astype(np.float16))


@pytest.mark.parametrize("m,n", [(20000, 3), (5000, 320), (301, 1283)])
@pytest.mark.parametrize("size", [1.0, 1e-5, 400.0, 2000.0, 3e38])
def test_dequantize_rounds_once(m, n, size):
    """fp16 results are the products' own roundings, bit for bit: an fp32 product that lands on the half between two fp16 values decides nothing
    (one value in 16000; `size` brings subnormal results and infinite ones in)."""
    from dynamicscaler_amd import ops
    d = dev()
    q = ints((m, n), m)
    s = torch.rand(m, generator=gen(n)) * size
    v = q.double() * s.double()[:, None]
    assert bool((once(v) != v.float().to(F16)).any()) or m * n < 10 ** 6 or size > 1e4              # there are such values among them
    assert torch.equal(ops.dequantize_rows_i8(q.to(d), s.to(d)).cpu(), once(v))
    assert torch.equal(ops.dequantize_rows_i8(q.to(d), s.to(d), dtype=F32).cpu(), v.float())


@pytest.mark.parametrize("m,n", [(400000, 5), (5000, 320), (1501, 1283), (100, 20011)])
@pytest.mark.parametrize("xt,rt", [(F32, F16), (F16, F16), (F16, F32), (F32, None)])
@pytest.mark.parametrize("size", [1.0, 2e-5, 300.0])
def test_norm_rounds_once(m, n, xt, rt, size):
    """The fp16 sum and the fp16 result are single roundings of the 64-bit ones.  The result's root is within 2^-44 of itself: values that close
    to a half between two fp16 values are left out (2^-40: one in 10^8)."""
    from dynamicscaler_amd import ops
    d = dev()
    x, g = row_inputs(m, n, m + 7, F32).mul(size).to(xt), (1.0 + 0.2 * normal((n,), n)) * size
    r = None if rt is None else normal((m, n), m, rt, size)
    h, t, root = rows_ref(x, r, g, 1e-6, True)
    y, back = ops.rmsnorm(x.to(d), g.to(d), residual=None if r is None else r.to(d))
    v = t * root
    sure = once(v * (1 + 2.0 ** -40)) == once(v * (1 - 2.0 ** -40))
    assert bool(((y.cpu() == once(v)) | ~sure).all()) and float(sure.float().mean()) > 0.999
    if rt is not None:
        assert torch.equal(back.cpu(), once(h) if rt == F16 else h.float())


@pytest.mark.parametrize("xt", [F16, F32])
def test_quantize_halves_go_to_even(xt):
    """Quotients that are exact halves (63.5 at x = max / 2; a row whose steps are whole numbers), and their neighbours one ulp away."""
    from dynamicscaler_amd import ops
    d = dev()
    rows = []
    for top in (1.0, 3.0, 127.0, 254.0, 381.0, 0.0999755859375, 1000.0, 2.0 ** -14 * 3):
        v = torch.zeros(64)
        v[0] = top
        for k in range(0, 31):
            v[2 * k + 1] = (2 * k + 1) * top / 254.0 * (-1 if k % 2 else 1)
        v[2] = top / 2
        rows.append(v)
    x = torch.stack(rows).to(xt)
    below, above = x.clone(), x.clone()
    below[:, 1:] = torch.nextafter(x[:, 1:], torch.zeros_like(x[:, 1:])) if xt == F32 else (x[:, 1:].float() * (1 - 2.0 ** -11)).to(xt)
    above[:, 1:] = torch.nextafter(x[:, 1:], torch.full_like(x[:, 1:], 1e4)) if xt == F32 else (x[:, 1:].float() * (1 + 2.0 ** -11 * 1.5)).to(xt)
    x = torch.cat([x, below, above])
    from fractions import Fraction
    q, _ = ops.quantize_rows_i8(x.to(d))
    for i in range(x.shape[0]):
        top = max(abs(Fraction(float(v))) for v in x[i])
        for j in range(x.shape[1]):
            assert int(q[i, j]) == round(Fraction(float(x[i, j])) * 127 / top), (i, j, float(x[i, j]))


@pytest.mark.parametrize("n", [8, 65, 320, 1283, 5120, 20000])
@pytest.mark.parametrize("xt", [F16, F32])
def test_rows_of_zeros_and_non_finite_rows(n, xt):
    from dynamicscaler_amd import ops
    d = dev()
    x, g = row_inputs(6, n, n, xt), 1.0 + 0.2 * normal((n,), n)
    x[1] = 0.0
    x[2, n // 2] = float("nan")
    x[3, n - 1] = float("inf")
    x[4, 0] = float("-inf")
    r = normal((6, n), 3, F32)
    r[1] = 0.0
    for res in (None, r):
        for q, scale in (ops.quantize_rows_i8(x.to(d)), ops.rmsnorm_i8(x.to(d), g.to(d), residual=None if res is None else res.to(d))[:2]):
            assert float(scale[1]) == 0.0 and not bool(q[1].any())
            assert bool(scale[2:5].isnan().all()) and not bool(q[2:5].any())
            assert bool(scale[[0, 5]].isfinite().all()) and bool((q[[0, 5]].abs().amax(dim=1) == 127).all())
        y, _ = ops.rmsnorm(x.to(d), g.to(d), residual=None if res is None else res.to(d))
        assert not bool(y[1].any()) and bool(y[2].isnan().all()) and bool(y[[0, 5]].isfinite().all())
        assert bool(y[3, n - 1].isnan()) and bool(y[4, 0].isnan()) and not bool(y[3, :n - 1].any()) and not bool(y[4, 1:].any())
    assert bool(ops.dequantize_rows_i8(q, scale)[2].isnan().all())
    bad = g.clone()
    bad[n // 3] = float("nan")                   # a NaN in gamma: every row's largest value is unknown
    q, scale, _ = ops.rmsnorm_i8(x[[0, 5]].to(d), bad.to(d))
    assert bool(scale.isnan().all()) and not bool(q.any())


@pytest.mark.parametrize("n", [64, 1283, 5120])
def test_norm_of_the_largest_and_smallest_values(n):
    """fp32 rows whose squares leave fp32 (1e30, 1e-30), fp16 rows of 65504 (their sum with the residual leaves fp16), subnormal rows."""
    from dynamicscaler_amd import ops
    d = dev()
    g = 1.0 + 0.2 * normal((n,), n)
    for scale, xt, rt in ((1e30, F32, F32), (1e-30, F32, F32), (1e-41, F32, None), (1e-7, F16, None)):
        x = (row_inputs(3, n, n, F32) * scale).to(xt)
        r = None if rt is None else (normal((3, n), 5) * scale).to(rt)
        h, t, root = rows_ref(x, r, g, 1e-6, True)
        q, s, back = ops.rmsnorm_i8(x.to(d), g.to(d), residual=None if r is None else r.to(d))
        check_rows_i8(q, s, t, root)
        y, _ = ops.rmsnorm(x.to(d), g.to(d), residual=None if r is None else r.to(d), out_dtype=F32)
        close(y, t * root, 5 * H32 * (t * root).abs() + 2.0 ** -148, F32)
    x = torch.full((2, n), 65504.0, dtype=F16)
    x[:, 1::2] *= -1
    h, t, root = rows_ref(x, x, g, 1e-6, True)
    q, s, back = ops.rmsnorm_i8(x.to(d), g.to(d), residual=x.to(d))
    check_rows_i8(q, s, t, root)
    assert bool(back.isinf().all())


@pytest.mark.parametrize("n", [5, 64, 320, 1283, 5120, 16384, 20011])
@pytest.mark.parametrize("gain", [1e-3, 1e-10, 0.0])
def test_norm_of_sums_beyond_fp32(n, gain):
    """x + residual leaves fp32 while its product with a small gamma does not: finite inputs, so the rows' 8 bits are the exact quotients (the fp32
    sum h is infinite there).  Rows of one sign, of both, of a cancelling pair and ordinary ones, for every kernel a row's length chooses."""
    from dynamicscaler_amd import ops
    d = dev()
    big = row_inputs(5, n, n, F32)
    g = (1.0 + 0.2 * normal((n,), n)) * gain
    x = big / big.abs().amax(dim=1, keepdim=True) * 3.3e38
    r = x.clone()
    x[1], r[1] = x[1].abs(), r[1].abs()
    r[2] = -x[2] * 0.9999                         # cancels: the sum is ordinary, its parts are not
    r[3, ::2] = -r[3, ::2]                        # every second sum is zero
    x[4], r[4] = big[4], 2 * big[4]               # an ordinary row between them
    h, t, root = rows_ref(x, r, g, 1e-6, True)
    q, s, back = ops.rmsnorm_i8(x.to(d), g.to(d), residual=r.to(d))
    check_rows_i8(q, s, t, root)
    over = h.abs() > torch.finfo(F32).max
    assert bool(over[:2].any()) and torch.equal(back.cpu().isinf(), over) and bool(s.isfinite().all())


@pytest.mark.parametrize("m,n,off", [(5, 320, 8), (5, 320, 3), (4, 641, 1), (3, 5120, 16), (2, 9001, 5)])
@pytest.mark.parametrize("xt,rt", [(F16, F16), (F16, F32), (F32, F32)])
def test_rows_strides_and_neighbours(m, n, off, xt, rt):
    from dynamicscaler_amd import ops
    d = dev()
    x, g, r = row_inputs(m, n, 3, xt), 1.0 + 0.2 * normal((n,), n), normal((m, n), 4, rt)

    def inside(t, fill):
        wide = torch.full((m + 2, n + 2 * off + 3), fill, dtype=t.dtype, device=d)
        wide[1:-1, off:off + n] = t.to(d)
        return wide, wide[1:-1, off:off + n]

    h, t, root = rows_ref(x, r, g, 1e-6, True)
    X, R = inside(x, 5.0)[1], inside(r, -7.0)[1]
    qw, q = inside(torch.zeros(m, n, dtype=torch.int8), 55)
    hw, hs = inside(torch.zeros(m, n, dtype=rt), 99.0)
    yw, y = inside(torch.zeros(m, n, dtype=xt), 33.0)
    scale = torch.zeros(m, device=d)
    ops.rmsnorm_i8(X, g.to(d), residual=R, sum_out=hs, out=q, scale=scale)
    check_rows_i8(q, scale, t, root)
    close(hs, h, H32 * h.abs(), rt)
    hs.fill_(0)
    ops.rmsnorm(X, g.to(d), residual=R, sum_out=hs, out=y)
    close(y, t * root, 5 * H32 * (t * root).abs(), xt)
    close(hs, h, H32 * h.abs(), rt)
    for wide, inner, fill in ((qw, q, 55), (hw, hs, 99.0), (yw, y, 33.0)):
        inner.fill_(fill)
        assert bool((wide == fill).all())
    ops.quantize_rows_i8(X, out=q, scale=scale)
    check_rows_i8(q, scale, x.double(), torch.ones(m, 1, dtype=torch.float64))
    ops.dequantize_rows_i8(q, scale, out=y)
    v = q.cpu().double() * scale.cpu().double()[:, None]
    close(y, v, H32 * v.abs(), xt)
    for wide, inner, fill in ((qw, q, 55), (yw, y, 33.0)):
        inner.fill_(fill)
        assert bool((wide == fill).all())


@pytest.mark.parametrize("m,n", [(3, 320), (2, 1283), (2, 6000), (1, 20000)])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_norm_in_place(m, n, dtype):
    """The sum over the residual, and y over x."""
    from dynamicscaler_amd import ops
    d = dev()
    x, g, r = row_inputs(m, n, 3, dtype), 1.0 + 0.2 * normal((n,), n), normal((m, n), 4, dtype)
    h, t, root = rows_ref(x, r, g, 1e-6, True)
    xd, rd = x.to(d), r.to(d)
    q, scale, back = ops.rmsnorm_i8(xd, g.to(d), residual=rd, sum_out=rd)
    assert back is rd
    check_rows_i8(q, scale, t, root)
    close(rd, h, H32 * h.abs(), dtype)
    rd = r.to(d)
    y, _ = ops.rmsnorm(xd, g.to(d), residual=rd, sum_out=rd, out=xd)
    close(xd, t * root, 5 * H32 * (t * root).abs(), dtype)
    close(rd, h, H32 * h.abs(), dtype)


@pytest.mark.parametrize("m,n", [(5000, 320), (2051, 1283), (1100, 5120), (1027, 9000), (300, 16384)])
def test_many_rows(m, n):
    """More rows than a launch has teams: a team's later rows, gamma kept between them; every row against the definition."""
    from dynamicscaler_amd import ops
    d = dev()
    x, g, r = row_inputs(m, n, 3, F16), 1.0 + 0.2 * normal((n,), n), normal((m, n), 4, F32)
    h, t, root = rows_ref(x, r, g, 1e-6, True)
    q, scale, back = ops.rmsnorm_i8(x.to(d), g.to(d), residual=r.to(d))
    check_rows_i8(q, scale, t, root)
    close(back, h, H32 * h.abs(), F32)
    q, scale = ops.quantize_rows_i8(x.to(d))
    check_rows_i8(q, scale, x.double(), torch.ones(m, 1, dtype=torch.float64))
    v = q.cpu().double() * scale.cpu().double()[:, None]
    close(ops.dequantize_rows_i8(q, scale), v, H32 * v.abs(), F16)


@pytest.mark.parametrize("m,n", [(5000, 320), (2051, 1283), (1100, 5120), (300, 16384)])
def test_many_rows_in_fp32(m, n):
    """fp32 rows, with and without an fp16 residual, more of them than a launch has teams."""
    from dynamicscaler_amd import ops
    d = dev()
    x, g, r = row_inputs(m, n, 5, F32), 1.0 + 0.2 * normal((n,), n), normal((m, n), 6, F16)
    one = torch.ones(m, 1, dtype=torch.float64)
    q, scale = ops.quantize_rows_i8(x.to(d))
    check_rows_i8(q, scale, x.double(), one)
    for res in (None, r):
        h, t, root = rows_ref(x, res, g, 1e-6, True)
        q, scale, back = ops.rmsnorm_i8(x.to(d), g.to(d), residual=None if res is None else res.to(d))
        check_rows_i8(q, scale, t, root)
        y, again = ops.rmsnorm(x.to(d), g.to(d), residual=None if res is None else res.to(d), out_dtype=F32)
        close(y, t * root, 5 * H32 * (t * root).abs(), F32)
        if res is not None:
            assert torch.equal(back.cpu(), once(h)) and torch.equal(again, back)


def test_more_rows_than_a_launch_has_threads_for():
    """70 million rows of three values: more workgroups than a grid takes, so each walks several."""
    from dynamicscaler_amd import ops
    d = dev()
    x = torch.randint(-2000, 2001, (70_000_000, 3), device=d, dtype=torch.int16, generator=torch.Generator(device=d).manual_seed(1)).to(F16)
    q, scale = ops.quantize_rows_i8(x)
    top = x.float().abs().amax(dim=1, keepdim=True)            # whole numbers below 2^11: 127 x and the quotient's halves are exact in fp32
    assert torch.equal(q.float(), torch.where(top > 0, torch.round(127 * x.float() / top), torch.zeros_like(top)))
    y = ops.dequantize_rows_i8(q, scale, dtype=F32)
    assert torch.equal(y, q.float() * scale[:, None])


def test_rows_of_nothing():
    from dynamicscaler_amd import ops
    d = dev()
    x = torch.empty((0, 320), dtype=F16, device=d)
    q, scale = ops.quantize_rows_i8(x)
    assert tuple(q.shape) == (0, 320) and tuple(scale.shape) == (0,)
    assert tuple(ops.dequantize_rows_i8(q, scale).shape) == (0, 320)
    assert tuple(ops.rmsnorm_i8(x, torch.ones(320, device=d), residual=x)[2].shape) == (0, 320)


# ------------------------------------------------------------------------------------------------ together
def feed_forward(p, x, stream):
    """norm -> GEGLU product -> quantisation -> product onto the residual stream, as a transformer block runs them."""
    from dynamicscaler_amd import ops
    q, s, stream = ops.rmsnorm_i8(x, p["g"], residual=stream)
    hidden = ops.gemm_i8(q, p["w1"], s, p["s1"], bias=p["b1"], epilogue=EPI["geglu"])
    q2, s2 = ops.quantize_rows_i8(hidden)
    return ops.gemm_i8(q2, p["w2"], s2, p["s2"], bias=p["b2"], residual=stream, out_dtype=stream.dtype), (q, s, stream, hidden, q2, s2)


def block(width, seed, d):
    from dynamicscaler_amd import ops
    w1, w2 = normal((8 * width, width), seed, scale=width ** -0.5), normal((width, 4 * width), seed + 1, scale=(4 * width) ** -0.5)
    p = {"g": (1.0 + 0.2 * normal((width,), seed + 2)).to(d), "b1": normal((8 * width,), seed + 3, scale=0.1).to(d), "b2": normal((width,), seed + 4, scale=0.1).to(d)}
    p["w1"], p["s1"] = ops.quantize_rows_i8(w1.to(d))
    p["w2"], p["s2"] = ops.quantize_rows_i8(w2.to(d))
    return p, w1, w2


@pytest.mark.parametrize("rows,width", [(1, 64), (77, 320), (1030, 320), (300, 640)])
@pytest.mark.parametrize("rt", [F16, F32])
def test_feed_forward_of_a_block(rows, width, rt):
    """Each link against its definition on the inputs it was given, and the whole near the same feed-forward on unquantised operands: a
    quantised operand is off by at most half a step (max / 254) of its row, uniformly spread, so a product of K terms of two such operands
    is off by about sqrt(K / 12) steps: with maxima of ~4 standard deviations 4 / 127 / sqrt(12) = 0.9 % of the operand per side.  Two
    sides, two products: 2 % of the branch expected, 4 % held."""
    d = dev()
    p, w1, w2 = block(width, 50, d)
    x, r = normal((rows, width), 1, F16), normal((rows, width), 2, rt, 2.0)
    out, (q, s, stream, hidden, q2, s2) = feed_forward(p, x.to(d), r.to(d))
    h, t, root = rows_ref(x, r, p["g"].cpu(), 1e-6, True)
    check_rows_i8(q, s, t, root)
    close(stream, h, H32 * h.abs(), rt)
    c = {k: v.cpu() for k, v in p.items()}
    close(hidden, *product_ref(q.cpu(), c["w1"], s.cpu(), c["s1"], c["b1"], None, "geglu"), F16)
    check_rows_i8(q2, s2, hidden.cpu().double(), torch.ones(rows, 1, dtype=torch.float64))
    close(out, *product_ref(q2.cpu(), c["w2"], s2.cpu(), c["s2"], c["b2"], stream.cpu(), "none"), rt)
    z = ((t * root) @ w1.double().t() + c["b1"].double()).view(rows, -1, 2, 32)
    f = (z[:, :, 0] * 0.5 * z[:, :, 1] * torch.erfc(-z[:, :, 1] / math.sqrt(2.0))).reshape(rows, -1) @ w2.double().t()
    branch = out.cpu().double() - stream.cpu().double() - c["b2"].double()
    assert float((branch - f).norm() / f.norm()) <= 0.04


@pytest.mark.parametrize("rows,width", [(1, 64), (77, 320), (300, 1280)])
def test_feed_forward_behind_a_layernorm(rows, width):
    """The chain of a block with a LayerNorm: its fp16 rows are quantised, every link against its definition on the inputs it was given."""
    from dynamicscaler_amd import ops
    d = dev()
    p, _, _ = block(width, 70, d)
    stream = normal((rows, width), 1, F32, 2.0).to(d)
    x = ops.layernorm(stream, p["g"], torch.zeros(width, device=d))
    q, s = ops.quantize_rows_i8(x)
    hidden = ops.gemm_i8(q, p["w1"], s, p["s1"], bias=p["b1"], epilogue=EPI["geglu"])
    q2, s2 = ops.quantize_rows_i8(hidden)
    before = stream.cpu().clone()
    ops.gemm_i8(q2, p["w2"], s2, p["s2"], bias=p["b2"], residual=stream, out=stream)
    one = torch.ones(rows, 1, dtype=torch.float64)
    check_rows_i8(q, s, x.cpu().double(), one)
    c = {k: v.cpu() for k, v in p.items()}
    close(hidden, *product_ref(q.cpu(), c["w1"], s.cpu(), c["s1"], c["b1"], None, "geglu"), F16)
    check_rows_i8(q2, s2, hidden.cpu().double(), one)
    close(stream, *product_ref(q2.cpu(), c["w2"], s2.cpu(), c["s2"], c["b2"], before, "none"), F32)


def test_feed_forward_in_a_graph_and_on_two_streams():
    """A captured block replayed between eager work, and two blocks at once on two streams: every result equals the eager one."""
    d = dev()
    p, _, _ = block(320, 50, d)
    xs = [normal((rows, 320), rows, F16).to(d) for rows in (200, 16)]
    rs = [normal((rows, 320), rows + 1, F32).to(d) for rows in (200, 16)]
    eager = [feed_forward(p, x, r)[0] for x, r in zip(xs, rs)]
    torch.cuda.synchronize()
    graphs = []
    for x, r in zip(xs, rs):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            feed_forward(p, x, r)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = feed_forward(p, x, r)[0]
        graphs.append((g, out))
    for turn in range(3):
        for (g, out), ref in zip(graphs, eager):
            out.zero_()
            g.replay()
            again = feed_forward(p, xs[turn % 2], rs[turn % 2])[0]
            torch.cuda.synchronize()
            assert torch.equal(out, ref) and torch.equal(again, eager[turn % 2])
    x0 = xs[0].clone()
    xs[0].copy_(x0 * 2)                              # new inputs in the captured buffers
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], feed_forward(p, xs[0], rs[0])[0])
    xs[0].copy_(x0)
    torch.cuda.synchronize()
    (a, w, sa, sw, b, _), _ = large_case(2057, 997, 1273, F16, None, "none")      # a call with a workspace and a large tile, captured
    from dynamicscaler_amd import ops
    ref = ops.gemm_i8(a, w, sa, sw, bias=b)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.gemm_i8(a, w, sa, sw, bias=b)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
        assert torch.equal(ops.gemm_i8(a, w, sa, sw, bias=b), ref)
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i] = feed_forward(p, xs[i], rs[i])[0]
    torch.cuda.synchronize()
    for got, ref in zip(outs, eager):
        assert torch.equal(got, ref)


def calls_that_allocate(d):
    """Each operator as a call without outputs, keyword arguments to come; the product with odd rows, which it lays out anew in a workspace."""
    from dynamicscaler_amd import ops
    (a, w, sa, sw, b, r), _ = large_case(2057, 997, 1273, F32, F32, "none")
    x, g, res = normal((301, 1283), 1, F16).to(d), normal((1283,), 2).to(d), normal((301, 1283), 3).to(d)
    q, s = ops.quantize_rows_i8(x)
    return {"product": lambda **kw: (ops.gemm_i8(a, w, sa, sw, bias=b, residual=r, out_dtype=F32, **kw),),
            "norm": lambda **kw: ops.rmsnorm(x, g, residual=res, **kw),
            "norm_i8": lambda **kw: ops.rmsnorm_i8(x, g, residual=res, **kw),
            "quantize": lambda **kw: ops.quantize_rows_i8(x, **kw),
            "dequantize": lambda **kw: (ops.dequantize_rows_i8(q, s, **kw),)}


@pytest.mark.parametrize("which", ["product", "norm", "norm_i8", "quantize", "dequantize"])
def test_outputs_of_a_call_on_a_named_stream_belong_to_it(which):
    """A block that the current stream gave back is still its own (kernels in flight may use it): the outputs of a call on another stream are
    other blocks, and come back to that stream.  The results are the same, captured ones too, and the current stream stays what it was."""
    d = dev()
    call = calls_that_allocate(d)[which]
    ref = call()
    side, here = torch.cuda.Stream(), torch.cuda.current_stream()
    torch.cuda.synchronize()
    blocks = [torch.empty_like(t) for t in ref]
    theirs = {t.data_ptr() for t in blocks}
    del blocks
    outs = call(stream=side.cuda_stream)
    assert torch.cuda.current_stream() == here
    side.synchronize()
    assert not theirs & {t.data_ptr() for t in outs}
    assert all(torch.equal(a, b) for a, b in zip(outs, ref))
    again = call(stream=here.cuda_stream)
    here.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, ref))
    mine = {t.data_ptr() for t in outs}
    del outs
    blocks = [torch.empty_like(t) for t in ref]
    assert not mine & {t.data_ptr() for t in blocks}
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        side.wait_stream(torch.cuda.current_stream())
        outs = call(stream=side.cuda_stream)
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        for t in outs:
            t.zero_()
        g.replay()
        eager = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(outs, ref, eager))


def test_products_with_a_workspace_on_two_streams():
    """Each call's workspace is its own stream's: two at once, the current stream's and a named one's, do not meet."""
    from dynamicscaler_amd import ops
    cases = [large_case(2057, 997, 1273, F16, None, "none", seed)[0] for seed in (1, 2)]
    refs = [ops.gemm_i8(a, w, sa, sw, bias=b) for a, w, sa, sw, b, _ in cases]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(8):
        for (a, w, sa, sw, b, _), stream in zip(cases, (None, side.cuda_stream)):
            outs.append(ops.gemm_i8(a, w, sa, sw, bias=b, stream=stream))
    torch.cuda.synchronize()
    for i, got in enumerate(outs):
        assert torch.equal(got, refs[i % 2])


@pytest.mark.parametrize("m,n,k", [(2057, 997, 1273), (2057, 1000, 1284), (1500, 1056, 4095)])
@pytest.mark.parametrize("flags", [0, 4, 2, 2 | 4 | 8])
def test_product_c_entry_without_a_workspace(m, n, k, flags):
    """The C entry with and without room for aligned copies, SiLU in front of a residual among the flags (the tensor front end's calls always
    bring the room that helps): the same bits, and right."""
    import ctypes as C
    from dynamicscaler_amd import _lib
    out_dtype, residual = (F32 if flags & 4 else F16), (F32 if flags & 8 else F16)
    act = "silu" if flags & 2 else "none"
    (a, w, sa, sw, b, r), (ref, before) = large_case(m, n, k, out_dtype, residual, act)
    lib, st, outs = _lib.load(), torch.cuda.current_stream().cuda_stream, []
    desc = _lib.GemmI8Desc(lda=k, ldw=k, ldc=n, ldr=n, M=m, N=n, K=k, epilogue=flags)
    need = lib.ds_gemm_i8_workspace_bytes(a.data_ptr(), w.data_ptr(), C.byref(desc))
    assert need > 0
    room = torch.empty(need, dtype=torch.uint8, device=a.device)
    for at, size in ((0, 0), (room.data_ptr(), need)):
        outs.append(torch.empty((m, n), dtype=out_dtype, device=a.device))
        assert lib.ds_gemm_i8(a.data_ptr(), w.data_ptr(), sa.data_ptr(), sw.data_ptr(), b.data_ptr(), r.data_ptr(), outs[-1].data_ptr(), C.byref(desc), at, size, st) == 0
    assert torch.equal(*outs)
    off = (outs[0].double() - ref).abs()
    assert float((off / (before + HALF[out_dtype] * (ref.abs() + before) + SUB[out_dtype])).max()) <= 1.0


@contextlib.contextmanager
def at_most(mib):
    """The allocator may take `mib` MiB more than what is held now, and gives nothing out of that (a pool of its own)."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (mib << 20)) / torch.cuda.get_device_properties(0).total_memory)
    try:
        with torch.cuda.use_mem_pool(torch.cuda.MemPool()):
            yield
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)


def test_outputs_that_do_not_fit_raise_as_everywhere():
    """torch.OutOfMemoryError, as the other operators' allocations do; the same call goes through once there is room."""
    from dynamicscaler_amd import ops
    d = dev()
    x, g = torch.ones((50000, 2048), dtype=F16, device=d), torch.ones(2048, device=d)
    q, s = ops.quantize_rows_i8(x)
    calls = [lambda: ops.gemm_i8(q, q[:2048], s, s[:2048]), lambda: ops.rmsnorm(x, g), lambda: ops.rmsnorm_i8(x, g), lambda: ops.quantize_rows_i8(x),
             lambda: ops.dequantize_rows_i8(q, s)]
    with at_most(16):
        for call in calls:
            with pytest.raises(torch.OutOfMemoryError):
                call()
    for call in calls:
        call()
    torch.cuda.synchronize()


def test_product_without_room_for_its_workspace():
    """The workspace only makes odd rows quicker: where it cannot be had the call reads them as they lie, with the same bits."""
    from dynamicscaler_amd import ops
    d = dev()
    a, w, sa, sw, b, _ = [None if t is None else t.to(d) for t in product_case(20057, 1997, 1273, 5)]
    ref = ops.gemm_i8(a, w, sa, sw, bias=b)
    out = torch.zeros_like(ref)
    with at_most(2):                              # (28 MB of copies)
        with pytest.raises(torch.OutOfMemoryError):
            torch.empty((20057 + 1997) * 1280, dtype=torch.int8, device=d)
        ops.gemm_i8(a, w, sa, sw, bias=b, out=out)
        torch.cuda.synchronize()
    assert torch.equal(out, ref)


def test_timing_hook_sees_the_product():
    from dynamicscaler_amd import ops
    seen = []

    def hook(name, flops, launch, info):
        seen.append((name, flops))
        launch()

    c = product_case(4, 64, 128, 2)
    ops.set_timing_hook(hook)
    try:
        got = run_product(c)
    finally:
        ops.set_timing_hook(None)
    assert seen == [("gemm_i8", 2.0 * 4 * 64 * 128)]
    close(got, *product_ref(*c, "none"), F16)
