"""The 8-bit operators and the token order on the GPU, against plain 64-bit restatements.

u = 2^-24 is half a step of fp32 relative to the value, 2^-8 half a step of bf16, 2^-4 of e4m3 (2^-10
below its smallest normal number). Tolerances count roundings:
* a row's sum of n squares is at most 32 terms in one thread and 10 in the tree, all positive: 42 u;
  with the mean, root, reciprocal and products v is within 21 + 11 = 32 u of its value
* swiglu: exp, 1 + exp, quotient and products within 16 u
* a scale is one division more, a code at most half a step of its type from v / s
* products: the integer sum is exact; conversion and two products are 3 u
* a sum of k products: (k + 1) u of the sum of the magnitudes; a dot product of H: (H / 32 + 16) u
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF = {torch.bfloat16: 2.0 ** -8, torch.float32: U}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import dsmoe
    return dsmoe


def rnd(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to("cuda").to(dtype)


def within(got, want, tol):
    d = (got.double() - want).abs()
    bad = ~(d <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float((d - tol).max()):.3g} over the tolerance"


def check_quant(q, s, v, fmt, rel, pow2=False):
    """Codes and scales of v (64-bit) with v itself known to ``rel``."""
    top = 448.0 if fmt == "fp8" else 127.0
    b = v.unflatten(-1, (-1, 128)) if fmt == "fp8" else v.unsqueeze(-2)
    sd = s.double().unsqueeze(-1) if fmt == "fp8" else s.double()[..., None, None]
    ref = b.abs().amax(-1, keepdim=True).clamp(min=1e-4) / top
    if pow2:
        assert bool((torch.frexp(s)[0] == 0.5).all())
        assert bool(((sd >= ref * (1 - rel)) & (sd < 2 * ref * (1 + rel))).all())
    else:
        within(sd, ref, ref * (rel + 2 * U))
    x = b / sd
    qd = q.float().double()
    qd = qd.unflatten(-1, (-1, 128)) if fmt == "fp8" else qd.unsqueeze(-2)
    step = torch.clamp(x.abs() * 2.0 ** -4, min=2.0 ** -10) if fmt == "fp8" else torch.full_like(x, 0.5)
    within(qd, x, step * (1 + 2 * U) + x.abs() * (rel + 4 * U))


def norm_ref(x, w, r, eps=1e-6):
    h = x.double()
    if r is not None:
        h = (x.float() + r.float()).to(x.dtype).double()
    return h, h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.double()


NORM_SHAPES = [("fp8", 1, 128), ("fp8", 1, 5120), ("fp8", 3, 1024), ("fp8", 33, 2304), ("fp8", 150, 8192), ("fp8", 5, 16384),
               ("int8", 1, 1), ("int8", 2, 7), ("int8", 1, 5120), ("int8", 65, 1040), ("int8", 9, 8191), ("int8", 4, 16384),
               ("int8", 5, 12345), ("int8", 301, 257), ("int8", 7, 4098), ("int8", 9, 16383), ("int8", 40, 9), ("int8", 33, 2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt,rows,n", NORM_SHAPES)
def test_rms_norm_quant(ops, fmt, rows, n, dtype):
    x, r, w = rnd(1, rows, n, dtype=dtype), rnd(2, rows, n, dtype=dtype, scale=3.0), 1 + 0.2 * rnd(3, n)
    got = ops.rms_norm_quant(x, w, r, fmt=fmt, normed=True)
    h, v = norm_ref(x, w, r)
    assert torch.equal(got.residual.double(), h)
    within(got.normed, v, v.abs() * (32 * U + BF[dtype]))
    check_quant(got.q, got.s, v, fmt, 32 * U)
    plain = ops.rms_norm_quant(x, w, fmt=fmt)
    assert plain.residual is None and plain.normed is None
    check_quant(plain.q, plain.s, norm_ref(x, w, None)[1], fmt, 32 * U)


@pytest.mark.parametrize("fmt,rows,n", [("fp8", 4096, 5120), ("int8", 2047, 1040), ("fp8", 1777, 8192), ("int8", 5000, 4104)])
def test_rms_norm_quant_many_rows(ops, fmt, rows, n):
    x, r, w = rnd(1, rows, n, dtype=torch.bfloat16), rnd(2, rows, n, dtype=torch.bfloat16, scale=3.0), 1 + 0.2 * rnd(3, n)
    x[rows - 1, 3] = float("nan")
    got = ops.rms_norm_quant(x, w, r, fmt=fmt, normed=True)
    h, v = norm_ref(x, w, r)
    last = slice(0, rows - 1)
    assert torch.equal(got.residual[last].double(), h[last]) and bool(torch.isnan(got.s[rows - 1]).all())
    within(got.normed[last], v[last], v[last].abs() * (32 * U + BF[torch.bfloat16]))
    check_quant(got.q[last], got.s[last], v[last], fmt, 32 * U)
    keep, keep_x = r.clone(), x.clone()
    again = ops.rms_norm_quant(keep_x, w, keep, fmt=fmt, inplace=True)
    assert torch.equal(keep[last], got.residual[last]) and torch.equal(again.s[last], got.s[last])
    one = ops.rms_norm_quant(x[:rows - 1], w, fmt=fmt)
    check_quant(one.q, one.s, norm_ref(x[last], w, None)[1], fmt, 32 * U)


@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,n", [(3, 17), (9, 24), (40, 31), (301, 1501), (200, 2050), (150, 6387), (5, 8195)])
def test_rms_norm_quant_odd_rows(ops, rows, n, dtype, wdtype):
    """Every offset of a row to 16 bytes, one and two chunks a thread, weights of both types."""
    x, r, w = rnd(126, rows, n, dtype=dtype), rnd(127, rows, n, dtype=dtype), (1 + 0.2 * rnd(128, n)).to(wdtype)
    got = ops.rms_norm_quant(x, w, r, fmt="int8", normed=True)
    h, v = norm_ref(x, w, r)
    assert torch.equal(got.residual.double(), h)
    within(got.normed, v, v.abs() * (32 * U + BF[dtype]))
    check_quant(got.q, got.s, v, "int8", 32 * U)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 2, 34, 255])
@pytest.mark.parametrize("n", [1, 2, 3, 5, 7, 9])
def test_rows_shorter_than_a_chunk(ops, rows, n, dtype):
    """Rows of a few values: many in one 16-byte chunk, the last ones less than a chunk before the end."""
    x, r, w = rnd(115, rows, n, dtype=dtype), rnd(116, rows, n, dtype=dtype), 1 + 0.2 * rnd(117, n)
    got = ops.rms_norm_quant(x, w, r, fmt="int8", normed=True)
    h, v = norm_ref(x, w, r)
    assert torch.equal(got.residual.double(), h)
    within(got.normed, v, v.abs() * (32 * U + BF[dtype]))
    check_quant(got.q, got.s, v, "int8", 32 * U)
    gu = rnd(118, rows, 2 * n, dtype=dtype, scale=4.0)
    q, s = ops.swiglu_quant(gu)
    check_quant(q, s, swiglu_ref(gu), "int8", 16 * U)


def test_rms_norm_quant_forms(ops):
    x, r, w = rnd(4, 2, 3, 256, dtype=torch.bfloat16), rnd(5, 2, 3, 256, dtype=torch.bfloat16), rnd(6, 256, dtype=torch.bfloat16)
    _, v = norm_ref(x, w, r, 0.1)
    got = ops.rms_norm_quant(x, w, r, eps=0.1)
    assert got.q.shape == (2, 3, 256) and got.s.shape == (2, 3, 2) and got.q.dtype == torch.float8_e4m3fn
    check_quant(got.q, got.s, v, "fp8", 32 * U)
    p2 = ops.rms_norm_quant(x, w, r, eps=0.1, scale_fmt="ue8m0")
    check_quant(p2.q, p2.s, v, "fp8", 32 * U, pow2=True)
    # transposed storage, a row range off 16-byte alignment, and the residual in place
    xt = x.transpose(0, 1).contiguous().transpose(0, 1)
    again = ops.rms_norm_quant(xt, w, r, eps=0.1)
    assert torch.equal(again.q.view(torch.uint8), got.q.view(torch.uint8)) and torch.equal(again.s, got.s)
    flat = torch.cat([x.new_zeros(1), x.flatten()])[1:].view(2, 3, 256)
    off = ops.rms_norm_quant(flat, w, r, eps=0.1)
    assert torch.equal(off.q.view(torch.uint8), got.q.view(torch.uint8))
    keep = r.clone()
    inp = ops.rms_norm_quant(x, w, keep, eps=0.1, inplace=True)
    assert inp.residual is keep and torch.equal(keep, got.residual) and torch.equal(inp.s, got.s)
    odd = torch.cat([r.new_zeros(1), r.flatten()])[1:].view(2, 3, 256)  # in place at an odd address
    i8, want = ops.rms_norm_quant(x, w, odd, fmt="int8", inplace=True), ops.rms_norm_quant(x, w, r, fmt="int8")
    assert torch.equal(odd, want.residual) and torch.equal(i8.q, want.q)
    odd = torch.cat([r.new_zeros(1), r.flatten()])[1:].view(2, 3, 256)
    f8 = ops.rms_norm_quant(x, w, odd, eps=0.1, inplace=True)
    assert f8.residual is odd and torch.equal(odd, got.residual) and torch.equal(f8.s, got.s)
    # one tensor as both terms
    twice = ops.rms_norm_quant(x, w, x, fmt="int8")
    check_quant(twice.q, twice.s, norm_ref(x, w, x)[1], "int8", 32 * U)


def test_written_tensors_are_known_to_autograd(ops):
    x, w = rnd(119, 3, 256), torch.ones(256, device="cuda")
    a, b, sa, sb = codes(120, 3, 64), codes(121, 256, 64), scales(122, 3), scales(123, 256)
    for r in (rnd(124, 3, 256), torch.zeros(769, device="cuda")[1:].view(3, 256)):
        leaf = rnd(125, 3, 256).requires_grad_()
        for write in (lambda: ops.rms_norm_quant(x, w, r, inplace=True), lambda: ops.int8_gemm(a, sa, b, sb, out=r)):
            y, before = (leaf * r).sum(), r._version
            write()
            assert r._version > before
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()
    with torch.inference_mode():
        r, out = rnd(124, 3, 256), torch.empty(3, 256, device="cuda")
        want = ops.int8_gemm(a, sa, b, sb)
    ops.rms_norm_quant(x, w, r, inplace=True)
    assert torch.equal(r, x + rnd(124, 3, 256)) and torch.equal(ops.int8_gemm(a, sa, b, sb, out=out), want)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_rms_norm_quant_special_rows(ops, fmt):
    x, w = rnd(7, 6, 256, dtype=torch.bfloat16), torch.ones(256, device="cuda")
    x[1] = 0.0
    x[2, 3], x[3, 200], x[4, 5] = float("nan"), float("inf"), float("-inf")
    got = ops.rms_norm_quant(x, w, fmt=fmt)
    vals = got.q.float().unflatten(-1, (-1, 128)) * got.s.unsqueeze(-1) if fmt == "fp8" else got.q.float() * got.s[:, None]
    ok = torch.tensor([0, 1, 5], device="cuda")
    _, v = norm_ref(x, w, None)
    check_quant(got.q[ok], got.s[ok], v[ok], fmt, 32 * U)
    assert not got.q[1].float().any() and bool(torch.isfinite(got.s[1]).all())
    assert bool(torch.isnan(vals[2:5]).all()) and bool(torch.isnan(got.s[2:5]).all())
    x[0, 7] = 3e30  # its square overflows: not a row of zeros
    big = ops.rms_norm_quant(x[:1], w, fmt=fmt, normed=True)
    assert bool(torch.isnan(big.s).all()) and bool(torch.isnan(big.normed).all())


def test_power_of_two_scales_at_their_borders(ops):
    x = torch.ones((1, 384), device="cuda")  # mean 1, eps 0: v is the weight, exactly
    w = torch.full((384,), 0.25, device="cuda")
    w[5], w[130], w[260] = 448.0, -3.5, 448.0 * (1 + 2.0 ** -23)
    got = ops.rms_norm_quant(x, w, eps=0.0, scale_fmt="ue8m0")
    assert got.s.tolist() == [[1.0, 2.0 ** -7, 2.0]]


def swiglu_ref(gu, wr=None, limit=10.0):
    g, u = gu.double().chunk(2, -1)
    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    h = g * torch.sigmoid(g) * u
    return h if wr is None else h * wr.double().unsqueeze(-1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt,rows,n", [("fp8", 1, 128), ("fp8", 48, 2048), ("fp8", 5, 2304), ("fp8", 3, 16384), ("int8", 1, 1),
                                        ("int8", 3, 7), ("int8", 48, 2048), ("int8", 5, 2049), ("int8", 200, 288),
                                        ("int8", 3, 16384), ("int8", 2, 9001), ("int8", 9, 16383), ("int8", 70, 5), ("int8", 33, 130),
                                        ("int8", 17, 1027)])
def test_swiglu_quant(ops, fmt, rows, n, dtype):
    gu, wr = rnd(8, rows, 2 * n, dtype=dtype, scale=4.0), rnd(9, rows).abs() + 0.1
    q, s = ops.swiglu_quant(gu, fmt=fmt)
    check_quant(q, s, swiglu_ref(gu), fmt, 16 * U)
    q, s = ops.swiglu_quant(gu, wr, limit=3.0, fmt=fmt)
    check_quant(q, s, swiglu_ref(gu, wr, 3.0), fmt, 17 * U)


@pytest.mark.parametrize("fmt,rows,n", [("fp8", 12283, 2048), ("int8", 6001, 4096), ("int8", 24001, 136), ("int8", 9001, 1000),
                                        ("fp8", 20000, 256)])
def test_swiglu_quant_many_rows(ops, fmt, rows, n):
    gu, wr = rnd(113, rows, 2 * n, dtype=torch.bfloat16, scale=4.0), rnd(114, rows)
    gu[rows - 1, 3] = float("nan")
    q, s = ops.swiglu_quant(gu, wr, fmt=fmt)
    check_quant(q[:-1], s[:-1], swiglu_ref(gu, wr)[:-1], fmt, 17 * U)
    assert bool(torch.isnan(s[-1]).any())


def test_swiglu_quant_special_values(ops):
    gu = rnd(10, 5, 512, dtype=torch.bfloat16)
    gu[0] = 0.0
    gu[1, 4], gu[2, 300] = float("nan"), float("nan")
    gu[3, 7], gu[3, 8] = float("inf"), float("-inf")   # gates: the limit, and silu(-inf)
    gu[4, 256 + 9], gu[4, 256 + 10] = float("inf"), float("-inf")
    q, s = ops.swiglu_quant(gu)
    assert not q[0].any() and bool(torch.isnan(s[1:3]).all())
    v = swiglu_ref(gu[4:])
    check_quant(q[4:], s[4:], v, "int8", 16 * U)
    assert bool(torch.isnan(s[3]))  # -inf * 0: the formula's value is NaN
    gu[3, 8] = -200.0
    gu[3, 256 + 8] = 2.0
    q, s = ops.swiglu_quant(gu[3:4])
    check_quant(q, s, swiglu_ref(gu[3:4]), "int8", 16 * U)
    q2, s2 = ops.swiglu_quant(gu[3:4], fmt="fp8", scale_fmt="ue8m0")
    check_quant(q2, s2, swiglu_ref(gu[3:4]), "fp8", 16 * U, pow2=True)


def codes(seed, *shape):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int8).to("cuda")


def scales(seed, *shape):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(shape, generator=g) + 0.1).to("cuda")


def product_tol(want, dtype):
    return want.abs() * (3 * U + (BF[dtype] if dtype != torch.float32 else 0.0))


GEMM_SHAPES = [(1, 1, 16), (1, 128, 128), (1, 4096, 5120), (3, 129, 48), (8, 512, 2048), (16, 127, 1040), (17, 300, 640),
               (32, 4096, 512), (33, 64, 4096), (64, 65, 144), (65, 257, 272), (100, 5120, 2048), (128, 1000, 5120),
               (255, 384, 384), (256, 256, 1024), (257, 130, 336), (700, 1111, 208), (1000, 4096, 256), (2500, 640, 2064)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", GEMM_SHAPES)
def test_int8_gemm(ops, m, n, k, dtype):
    a, b, sa, sb = codes(11, m, k), codes(12, n, k), scales(13, m), scales(14, n)
    got = ops.int8_gemm(a, sa, b, sb, out_dtype=dtype)
    want = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()
    assert got.dtype == dtype and got.shape == (m, n)
    within(got, want, product_tol(want, dtype))


def test_int8_gemm_extremes(ops):
    # the largest sums: -128 * -128 * 131056 = 2147221504 fits in 32 bits
    k = 131056
    a, b = torch.full((3, k), -128, dtype=torch.int8, device="cuda"), torch.full((130, k), -128, dtype=torch.int8, device="cuda")
    b[1::2] = 127
    one = torch.ones(130, device="cuda")
    got = ops.int8_gemm(a, one[:3], b, one, out_dtype=torch.float32)
    want = torch.where(torch.arange(130, device="cuda") % 2 == 0, 16384.0 * k, -16256.0 * k).double().expand(3, -1)
    within(got, want, want.abs() * U)


def test_int8_gemm_forms(ops):
    a, b, sa, sb = codes(15, 2, 3, 96), codes(16, 40, 96), scales(17, 2, 3), scales(18, 40)
    want = ops.int8_gemm(a, sa, b, sb)
    assert want.dtype == torch.float32 and want.shape == (2, 3, 40)
    wide = codes(15, 40, 192)
    wide[:, :96] = b  # a view with a longer row, and one at an odd address
    odd = torch.cat([a.new_zeros(3), a.flatten()])[3:].view(2, 3, 96)
    assert torch.equal(ops.int8_gemm(odd, sa, wide[:, :96], sb), want)
    out = torch.full((2, 3, 40), 7.0, device="cuda", dtype=torch.bfloat16)
    assert ops.int8_gemm(a, sa, b, sb, out=out) is out and torch.equal(out, want.to(torch.bfloat16))
    assert ops.int8_gemm(a[:0], sa[:0], b, sb).shape == (0, 3, 40)
    torch.set_default_dtype(torch.bfloat16)
    try:
        assert ops.int8_gemm(a, sa, b, sb).dtype == torch.bfloat16
    finally:
        torch.set_default_dtype(torch.float32)
    nan = sa.clone()
    nan[0, 1] = float("nan")  # a token without a scale stays one
    got = ops.int8_gemm(a, nan, b, sb)
    assert bool(torch.isnan(got[0, 1]).all()) and torch.equal(got[1], want[1])


def group_offsets(counts):
    return torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device="cuda")


GROUPS = [([1], 128, 128, 0), ([0, 0, 5], 64, 48, 0), ([3, 0, 1, 2, 0], 200, 272, 4), ([0, 0, 0], 130, 64, 6),
          ([17, 300, 0, 64, 1], 257, 208, 0), ([70] * 9, 384, 1024, 3), ([0] * 500 + [1] * 48 + [0] * 476, 32, 80, 0),
          ([600, 2, 0, 33, 257], 130, 400, 11), ([1, 2, 3, 4] * 12, 512, 512, 0), ([16] * 30, 96, 2048, 0)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts,n,k,tail", GROUPS)
def test_int8_grouped_gemm(ops, counts, n, k, tail, dtype):
    rows, e = sum(counts) + tail, len(counts)
    a, b, sa, sb = codes(19, rows, k), codes(20, e, n, k), scales(21, rows), scales(22, e, n)
    out = torch.full((rows, n), float("nan"), dtype=dtype, device="cuda")
    ops.int8_grouped_gemm(a, sa, b, sb, group_offsets(counts), out=out)
    at = 0
    for i, c in enumerate(counts):
        if c:
            want = (a[at:at + c].double() @ b[i].double().T) * sa[at:at + c].double()[:, None] * sb[i].double()
            within(out[at:at + c], want, product_tol(want, dtype))
        at += c
    assert not out[at:].any()


# more tiles than the pairs of CTAs of the GPU, of one and of two halves; tails: rows behind the last group
BIG_GROUPS = [([3000, 1, 2000, 0, 2999], 2100, 272, 0), ([1, 5000, 300], 4096, 16, 0), ([700, 513, 0, 33, 4000, 90], 3000, 640, 77),
              ([257] * 16, 1030, 144, 0), ([12000], 700, 48, 0), ([200, 4000, 1, 1500], 4100, 1040, 6000), ([40, 9], 4096, 64, 8000),
              ([0, 0, 0], 1500, 32, 9000), ([129] * 70, 640, 16, 1), ([1000, 31] * 12, 2304, 208, 0)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts,n,k,tail", BIG_GROUPS)
def test_int8_grouped_gemm_many_tiles(ops, counts, n, k, tail, dtype):
    test_int8_grouped_gemm(ops, counts, n, k, tail, dtype)


# rows, n, k, experts: from one row to thousands, few and many K blocks, every width of tile and split of K
SPREAD_GROUPS = [(1, 96, 1136, 2), (405, 700, 16, 40), (176, 257, 144, 40), (34, 130, 592, 40), (32, 96, 944, 40), (912, 700, 16, 40),
                 (43, 400, 496, 40), (35, 96, 1568, 40), (293, 257, 144, 40), (86, 130, 1312, 40), (75, 257, 928, 8),
                 (1391, 1500, 400, 5), (1947, 130, 1312, 40), (456, 121, 2960, 6), (324, 155, 1168, 6), (1437, 81, 3680, 146)]


@pytest.mark.parametrize("skew", [0.0, 1.1, 4.0])
@pytest.mark.parametrize("rows,n,k,e", SPREAD_GROUPS)
def test_int8_grouped_gemm_spreads(ops, rows, n, k, e, skew):
    g = torch.Generator().manual_seed(rows)
    p = torch.arange(1, e + 1, dtype=torch.float64)[torch.randperm(e, generator=g)] ** -skew
    counts = torch.bincount(torch.multinomial(p, rows, replacement=True, generator=g), minlength=e).tolist()
    test_int8_grouped_gemm(ops, counts, n, k, 0 if skew else 5, torch.bfloat16 if skew else torch.float32)


def test_int8_grouped_gemm_many_tiles_at_once(ops):
    """Two streams and a graph of calls in a row; offsets that describe no groups in the same shapes."""
    sets = []
    for i, counts in enumerate(([3000, 1, 2000, 0, 2999], [0, 8000, 0, 0, 0], [1, 2, 3, 4, 100])):
        off = group_offsets(counts)
        t = codes(130 + i, 8000, 272), scales(131 + i, 8000), codes(132 + i, 5, 2100, 272), scales(133 + i, 5, 2100), off
        sets.append((t, ops.int8_grouped_gemm(*t)))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            got.append(ops.int8_grouped_gemm(*sets[i % 3][0]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, sets[i % 3][1]) for i, g in enumerate(got))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = [ops.int8_grouped_gemm(*sets[i % 3][0]) for i in range(7)]
    for _ in range(3):
        for o in out:
            o.fill_(7.0)
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, sets[i % 3][1]) for i, o in enumerate(out))
    (a, sa, b, sb, _), _ = sets[0]
    for bad in ([0, 5, 3, 8, 8, 8], [0, 1, 2, 3, 4, 8001], [1, 1, 1, 1, 1, 8000]):
        assert bool(torch.isnan(ops.int8_grouped_gemm(a, sa, b, sb, torch.tensor(bad, dtype=torch.int32, device="cuda"))).all()), bad


def test_int8_grouped_gemm_bad_offsets(ops):
    a, b, sa, sb = codes(23, 8, 64), codes(24, 3, 40, 64), scales(25, 8), scales(26, 3, 40)
    for bad in ([0, 5, 3, 8], [1, 2, 3, 8], [0, 4, 6, 9], [0, -1, 4, 8], [-5, 0, 0, 0], [0, 2 ** 30, 2 ** 31 - 1, 8]):
        out = ops.int8_grouped_gemm(a, sa, b, sb, torch.tensor(bad, dtype=torch.int32, device="cuda"))
        assert bool(torch.isnan(out).all()), bad


# ------------------------------------------------------------------ tokens

def choices(seed, P, k, E, drop=0.0, skew=True):
    g = torch.Generator().manual_seed(seed)
    p = torch.arange(1, E + 1, dtype=torch.float64) ** (-1.1 if skew else 0.0)
    idx = torch.multinomial(p, P * k, replacement=True, generator=g).view(P, k)  # repeated experts within a token too
    idx[torch.rand((P, k), generator=g) < drop] = -1
    return idx.cuda()


def order_ref(idx, E):
    P, k = idx.shape
    flat = idx.flatten().cpu()
    pos = torch.full((P * k,), -1, dtype=torch.int32)
    src = torch.full((P * k,), -1, dtype=torch.int32)
    off, at = [0], 0
    for e in range(E):
        hit = torch.nonzero(flat == e).flatten()
        pos[hit] = torch.arange(at, at + len(hit), dtype=torch.int32)
        src[at:at + len(hit)] = hit.int()
        at += len(hit)
        off.append(at)
    return pos.view(P, k).cuda(), src.cuda(), torch.tensor(off, dtype=torch.int32).cuda()


ORDERS = [(1, 1, 1, 0.0), (1, 6, 384, 0.0), (8, 6, 384, 0.0), (5, 3, 128, 0.4), (33, 8, 7, 0.1), (2, 64, 1024, 0.0),
          (700, 6, 384, 0.2), (683, 6, 384, 0.0), (4099, 1, 1024, 0.0), (20000, 3, 60, 0.1), (9, 2, 5, 1.0), (43691, 6, 1, 0.0)]


@pytest.mark.parametrize("P,k,E,drop", ORDERS)
def test_sort_tokens(ops, P, k, E, drop):
    idx = choices(27, P, k, E, drop)
    for got, want in zip(ops.sort_tokens(idx, E), order_ref(idx, E)):
        assert torch.equal(got, want)
    wild = idx.clone()
    wild[idx == -1] = E + 5  # any number outside is a dropped choice
    wild[0, 0] = -(2 ** 62)
    keep = idx.clone()
    keep[0, 0] = -1
    for got, want in zip(ops.sort_tokens(wild, E), order_ref(keep, E)):
        assert torch.equal(got, want)


ROWS = [(1, 6, 384, 5120, 0.0), (8, 6, 384, 5120, 0.0), (5, 3, 12, 33, 0.4), (33, 8, 7, 1024, 0.1), (3, 64, 1024, 8, 0.0),
        (300, 6, 384, 520, 0.2), (9, 2, 5, 1, 1.0), (257, 1, 3, 4100, 0.0)]


@pytest.mark.parametrize("P,k,E,H,drop", ROWS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tokens_round_trip_and_gradients(ops, P, k, E, H, drop, dtype):
    idx = choices(28, P, k, E, drop)
    order = ops.sort_tokens(idx, E)
    n, live = P * k, int(order.offsets[-1])
    x, ys = rnd(29, P, H, dtype=dtype).requires_grad_(), rnd(30, n, H, dtype=dtype).requires_grad_()
    wt = rnd(31, P, k).requires_grad_()
    dxs, dy = rnd(32, n, H, dtype=dtype), rnd(33, P, H, dtype=dtype)
    xs, y = ops.dispatch_tokens(x, order), ops.combine_tokens(ys, order, wt)
    dx, dys, dwt = torch.autograd.grad((xs, y), (x, ys, wt), (dxs, dy))
    hit, pos = (order.pos >= 0), order.pos.long().clamp(min=0)
    want = torch.zeros((n, H), dtype=dtype, device="cuda")
    want[order.pos[hit].long()] = x.detach().repeat_interleave(k, 0)[hit.flatten()]
    assert torch.equal(xs, want) and not xs[live:].any()
    picked = torch.where(hit[..., None], ys.detach().double()[pos], 0.0)
    w64, half = wt.detach().double()[..., None], BF[dtype]
    want, mag = (picked * w64).sum(1), (picked * w64).abs().sum(1)
    within(y, want, mag * (k + 1) * U + want.abs() * half * (1 + U) + mag * (k + 1) * U * half)
    back = torch.where(hit[..., None], dxs.double()[pos], 0.0)
    within(dx, back.sum(1), back.abs().sum(1) * (k + 1) * U * (1 + half) + back.sum(1).abs() * half)
    want = torch.zeros((n, H), dtype=torch.float64, device="cuda")
    want[order.pos[hit].long()] = (dy.double().unsqueeze(1) * w64)[hit]
    within(dys, want, want.abs() * (half + U) * (1 + U))
    want, mag = (picked * dy.double().unsqueeze(1)).sum(-1), (picked * dy.double().unsqueeze(1)).abs().sum(-1)
    within(dwt, want, mag * (H / 32 + 16) * U)
    # without weights, and one gradient alone
    y1 = ops.combine_tokens(ys, order)
    (d1,) = torch.autograd.grad(y1, ys, dy)
    assert torch.equal(d1[:live], dy.repeat_interleave(k, 0)[order.src[:live].long()]) and not d1[live:].any()
    (dw,) = torch.autograd.grad(ops.combine_tokens(ys.detach(), order, wt), wt, dy)
    assert torch.equal(dw, dwt)
    (dz,) = torch.autograd.grad(ops.combine_tokens(ys, order, wt.detach()), ys, dy)
    assert torch.equal(dz, dys)


def test_gradients_against_differences(ops):
    """Small whole numbers: every product and sum is exact in fp32, so differences are too."""
    g = torch.Generator().manual_seed(34)
    whole = lambda *s: torch.randint(-4, 5, s, generator=g).float().cuda()
    idx = choices(35, 6, 3, 4, 0.2)
    order = ops.sort_tokens(idx, 4)
    x, ys, wt = whole(6, 20).requires_grad_(), whole(18, 20).requires_grad_(), whole(6, 3).requires_grad_()
    a, b = whole(18, 20), whole(6, 20)
    f = lambda x, ys, wt: float((ops.dispatch_tokens(x, order) * a).sum() + (ops.combine_tokens(ys, order, wt) * b).sum())
    loss = (ops.dispatch_tokens(x, order) * a).sum() + (ops.combine_tokens(ys, order, wt) * b).sum()
    grads = torch.autograd.grad(loss, (x, ys, wt))
    with torch.no_grad():
        for i, gr in enumerate(grads):
            d = whole(*gr.shape)
            args = [x, ys, wt]
            up, dn = list(args), list(args)
            up[i], dn[i] = args[i] + d, args[i] - d
            assert f(*up) - f(*dn) == 2 * float((gr * d).sum())


def test_tokens_non_finite_and_broadcast(ops):
    idx = torch.tensor([[0, 1], [1, -1], [-1, -1]], device="cuda")
    order = ops.sort_tokens(idx, 2)
    ys = torch.ones((6, 16), device="cuda")
    ys[order.offsets[-1]:] = float("nan")  # rows that belong to nobody are not read
    wt = torch.ones((3, 2), device="cuda")
    wt[1, 1] = wt[2, 0] = float("inf")     # nor are the weights of dropped choices
    wt.requires_grad_()
    y = ops.combine_tokens(ys, order, wt)
    assert torch.equal(y, torch.tensor([2.0, 1.0, 0.0], device="cuda")[:, None].expand(3, 16))
    (dwt,) = torch.autograd.grad(y.sum(), wt)  # an expanded gradient
    assert torch.equal(dwt, torch.tensor([[16.0, 16.0], [16.0, 0.0], [0.0, 0.0]], device="cuda"))
    x = torch.randn(1, 16, device="cuda").requires_grad_()
    xs = ops.dispatch_tokens(x.expand(3, 16), order)
    (dx,) = torch.autograd.grad(xs.sum(), x)   # the broadcast token's gradient sums over its three rows
    assert torch.equal(dx, torch.full((1, 16), 3.0, device="cuda"))


@pytest.mark.parametrize("width", [16, 48, 5120, 7, 1])
@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn, torch.float64])
def test_dispatch_quantized_rows(ops, width, dtype):
    idx = choices(36, 40, 4, 9, 0.3)
    order = ops.sort_tokens(idx, 9)
    x = rnd(37, 40, width, scale=20.0).to(dtype)
    s = scales(38, 40)
    xs, ss = ops.dispatch_tokens(x, order, s)
    live, src = int(order.offsets[-1]), order.src.long()
    byt = lambda t: t.contiguous().view(torch.uint8)
    assert torch.equal(byt(xs[:live]), byt(x)[src[:live] // 4]) and torch.equal(ss[:live], s[src[:live] // 4])
    assert not byt(xs[live:]).any() and not ss[live:].any()
    assert torch.equal(byt(ops.dispatch_tokens(x, order)), byt(xs))


def test_empty_batches(ops):
    order = ops.sort_tokens(torch.empty((0, 6), dtype=torch.int64, device="cuda"), 5)
    assert order.pos.shape == (0, 6) and order.src.shape == (0,) and not order.offsets.any() and len(order.offsets) == 6
    x = torch.empty((0, 32), device="cuda", requires_grad=True)
    xs = ops.dispatch_tokens(x, order)
    y = ops.combine_tokens(xs, order, torch.empty((0, 6), device="cuda"))
    (dx,) = torch.autograd.grad(y.sum(), x)
    assert y.shape == xs.shape == dx.shape == (0, 32)
    b, sb = codes(39, 5, 16, 32), scales(40, 5, 16)
    assert ops.int8_grouped_gemm(codes(41, 0, 32), scales(42, 0), b, sb, order.offsets).shape == (0, 16)
    w = torch.ones(128, device="cuda")
    q, s, _, _ = ops.rms_norm_quant(torch.empty((0, 128), device="cuda"), w)
    assert q.shape == (0, 128) and s.shape == (0, 1)
    assert ops.swiglu_quant(torch.empty((0, 256), device="cuda"))[1].shape == (0,)


def test_offsets_past_32_bits(ops):
    """Tensors of more than 2^31 values: the last rows are those of a small call on the same rows."""
    byt = lambda t: t.contiguous().view(torch.uint8)
    rows, n = 132000, 16383
    x = torch.zeros((rows, n), dtype=torch.bfloat16, device="cuda")
    x[-3:] = rnd(140, 3, n, dtype=torch.bfloat16)
    w = 1 + 0.2 * rnd(141, n)
    got, want = ops.rms_norm_quant(x, w, x, fmt="int8"), ops.rms_norm_quant(x[-3:].clone(), w, x[-3:].clone(), fmt="int8")
    check_quant(got.q[-3:], got.s[-3:], norm_ref(x[-3:], w, x[-3:])[1], "int8", 32 * U)
    assert torch.equal(got.residual[-3:], want.residual) and not got.q[:-3].any()
    del got
    half = x.view(-1)[:rows * n // 2 // 8191 * 8191 * 2].view(-1, 2 * 8191)
    half[-1] = rnd(142, 2 * 8191, dtype=torch.bfloat16)
    q, s = ops.swiglu_quant(half)
    q1, s1 = ops.swiglu_quant(half[-1:].clone())
    assert torch.equal(q[-1:], q1) and torch.equal(s[-1:], s1)
    del q, s, half
    x[-3:] = rnd(140, 3, n, dtype=torch.bfloat16)
    idx = torch.zeros((rows, 1), dtype=torch.int64, device="cuda")
    idx[-2] = 1  # the last row of all, the others in order
    order = ops.sort_tokens(idx, 2)
    xs = ops.dispatch_tokens(x, order)
    assert torch.equal(xs[-1], x[-2]) and torch.equal(xs[-2], x[-1])
    assert torch.equal(ops.combine_tokens(xs, order)[-3:], x[-3:])
    dy = xs.clone().requires_grad_()
    wt = torch.ones((rows, 1), device="cuda", requires_grad=True)
    ops.combine_tokens(dy, order, wt).backward(x)
    assert torch.equal(dy.grad[-2:], xs[-2:])
    within(wt.grad[-3:, 0], (x[-3:].double() ** 2).sum(-1), (x[-3:].double() ** 2).sum(-1) * (n / 32 + 16) * U)
    del x, xs, dy
    m, k = 290000, 48
    a, sa, b, sb = codes(143, m, k), scales(144, m), codes(145, 2, 8191, k), scales(146, 2, 8191)
    out = ops.int8_gemm(a, sa, b[0], sb[0], out_dtype=torch.bfloat16)
    assert torch.equal(byt(out[-5:]), byt(ops.int8_gemm(a[-5:], sa[-5:], b[0], sb[0], out_dtype=torch.bfloat16)))
    off = torch.tensor([0, m - 7, m - 2], dtype=torch.int32, device="cuda")
    ops.int8_grouped_gemm(a, sa, b, sb, off, out=out)
    assert torch.equal(out[-7:-2], ops.int8_gemm(a[-7:-2], sa[-7:-2], b[1], sb[1], out_dtype=torch.bfloat16)) and not out[-2:].any()


def test_refusals(ops):
    x, w = rnd(43, 4, 256, dtype=torch.bfloat16), torch.ones(256, device="cuda")
    for bad, err in ((lambda: ops.rms_norm_quant(x.half(), w), TypeError), (lambda: ops.rms_norm_quant(x, w[:128]), ValueError),
                     (lambda: ops.rms_norm_quant(x, w, x.float()), TypeError), (lambda: ops.rms_norm_quant(x, w, x[:2]), ValueError),
                     (lambda: ops.rms_norm_quant(x[:, :200], w[:200]), ValueError), (lambda: ops.rms_norm_quant(x, w, fmt="fp4"), ValueError),
                     (lambda: ops.rms_norm_quant(x, w, fmt="int8", scale_fmt="ue8m0"), ValueError),
                     (lambda: ops.rms_norm_quant(x, w, inplace=True), ValueError), (lambda: ops.rms_norm_quant(x, w.cpu()), ValueError),
                     (lambda: ops.rms_norm_quant(x, w.clone().requires_grad_()), ValueError),
                     (lambda: ops.rms_norm_quant(x, w, x.t().contiguous().t(), inplace=True), ValueError),
                     (lambda: ops.rms_norm_quant(rnd(1, 1, 16512), torch.ones(16512, device="cuda")), ValueError),
                     (lambda: ops.swiglu_quant(x[:, :255]), ValueError), (lambda: ops.swiglu_quant(x, limit=0.0), ValueError),
                     (lambda: ops.swiglu_quant(x, torch.ones(3, device="cuda")), ValueError),
                     (lambda: ops.swiglu_quant(x.clone().requires_grad_()), ValueError),
                     (lambda: ops.swiglu_quant(x[:, :200], fmt="fp8"), ValueError)):
        with pytest.raises(err):
            bad()
    a, b, sa, sb = codes(44, 4, 64), codes(45, 8, 64), scales(46, 4), scales(47, 8)
    off = group_offsets([4])
    for bad, err in ((lambda: ops.int8_gemm(a.float(), sa, b, sb), TypeError), (lambda: ops.int8_gemm(a[:, :40], sa, b[:, :40], sb), ValueError),
                     (lambda: ops.int8_gemm(a, sa, b[:, :48], sb), ValueError), (lambda: ops.int8_gemm(a, sa[:3], b, sb), ValueError),
                     (lambda: ops.int8_gemm(a, sa.double(), b, sb), TypeError), (lambda: ops.int8_gemm(a, sa, b, sb, torch.float16), TypeError),
                     (lambda: ops.int8_gemm(a, sa, b[None], sb), ValueError),
                     (lambda: ops.int8_gemm(a, sa, b, sb, out=torch.empty(4, 9, device="cuda")), ValueError),
                     (lambda: ops.int8_gemm(a, sa, b, sb, torch.bfloat16, torch.empty(4, 8, device="cuda")), TypeError),
                     (lambda: ops.int8_gemm(a, sa.clone().requires_grad_(), b, sb), ValueError),
                     (lambda: ops.int8_grouped_gemm(a, sa, b, sb, off), ValueError),
                     (lambda: ops.int8_grouped_gemm(a, sa, b[None], sb[None], off.long()), TypeError),
                     (lambda: ops.int8_grouped_gemm(a, sa, b[None], sb[None], off[:1]), ValueError),
                     (lambda: ops.int8_grouped_gemm(a, sa, b[None].expand(1025, 8, 64), sb[None].expand(1025, 8), off), ValueError)):
        with pytest.raises(err):
            bad()
    idx = choices(48, 4, 2, 3)
    order = ops.sort_tokens(idx, 3)
    for bad, err in ((lambda: ops.sort_tokens(idx.int(), 3), TypeError), (lambda: ops.sort_tokens(idx, 0), ValueError),
                     (lambda: ops.sort_tokens(idx, 1025), ValueError), (lambda: ops.sort_tokens(idx[:, :0], 3), ValueError),
                     (lambda: ops.dispatch_tokens(x[:3], order), ValueError), (lambda: ops.combine_tokens(x, order), ValueError),
                     (lambda: ops.combine_tokens(rnd(1, 8, 4).half(), order), TypeError),
                     (lambda: ops.combine_tokens(rnd(1, 8, 4), order, torch.ones(4, 3, device="cuda")), ValueError),
                     (lambda: ops.combine_tokens(rnd(1, 8, 4), order, torch.ones(4, 2, device="cuda").double()), TypeError),
                     (lambda: ops.dispatch_tokens(x, order, torch.ones(3, device="cuda")), ValueError),
                     (lambda: ops.dispatch_tokens(x.clone().requires_grad_(), order, torch.ones(4, device="cuda")), ValueError),
                     (lambda: ops.dispatch_tokens(x.double().requires_grad_(), order), TypeError)):
        with pytest.raises(err):
            bad()


# ------------------------------------------------------------------ streams, graphs, the operators in a row

def one_of_each(ops, t):
    order = ops.sort_tokens(t["idx"], 9)
    n = ops.rms_norm_quant(t["x"], t["w"], t["r"], fmt="int8", normed=True)
    xs, ss = ops.dispatch_tokens(n.q, order, n.s)
    gu = ops.int8_grouped_gemm(xs, ss, t["w13"], t["s13"], order.offsets, out_dtype=torch.bfloat16)
    q, s = ops.swiglu_quant(gu)
    ys = ops.int8_grouped_gemm(q, s, t["w2"], t["s2"], order.offsets, out_dtype=torch.bfloat16)
    return [n.q, n.s, n.residual, n.normed, order.pos, order.offsets, xs, gu, q, s, ys, ops.combine_tokens(ys, order, t["wt"]),
            ops.int8_gemm(n.q, n.s, t["w13"][0], t["s13"][0])]


def one_inputs(seed):
    return {"idx": choices(seed, 37, 3, 9, 0.1), "x": rnd(seed + 1, 37, 256, dtype=torch.bfloat16),
            "r": rnd(seed + 2, 37, 256, dtype=torch.bfloat16), "w": 1 + 0.1 * rnd(seed + 3, 256), "w13": codes(seed + 4, 9, 256, 256),
            "s13": scales(seed + 5, 9, 256) * 1e-3, "w2": codes(seed + 6, 9, 256, 128), "s2": scales(seed + 7, 9, 256),
            "wt": scales(seed + 8, 37, 3)}


def same(got, want):
    return all(torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)) for a, b in zip(got, want))


def test_streams_graphs_and_repeats(ops):
    t, other = one_inputs(50), one_inputs(70)
    want, want2 = one_of_each(ops, t), one_of_each(ops, other)
    assert same(one_of_each(ops, t), want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):  # two streams at once: nothing is shared between calls
        with torch.cuda.stream(streams[i % 2]):
            got.append(one_of_each(ops, t if i % 2 == 0 else other))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert same(g, want if i % 2 == 0 else want2)
    graphs = []
    for src in (t, other):
        g = torch.cuda.CUDAGraph()
        static = {k: v.clone() for k, v in src.items()}
        with torch.cuda.graph(g):
            out = one_of_each(ops, static)
        graphs.append((g, static, out))
    for _ in range(3):
        for g, _, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert same(graphs[0][2], want) and same(graphs[1][2], want2)
    for k, v in other.items():
        graphs[0][1][k].copy_(v)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert same(graphs[0][2], want2)


def test_backward_in_a_graph(ops):
    idx = choices(90, 20, 3, 7, 0.1)
    leaf = lambda seed, *s: rnd(seed, *s).requires_grad_()
    x, ys, wt = leaf(91, 20, 64), leaf(92, 60, 64), leaf(93, 20, 3)
    dxs, dy = rnd(94, 60, 64), rnd(95, 20, 64)

    def step():
        order = ops.sort_tokens(idx, 7)
        out = (ops.dispatch_tokens(x, order), ops.combine_tokens(ys, order, wt))
        return torch.autograd.grad(out, (x, ys, wt), (dxs, dy))

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_backward_capture_refused_beside_a_live_eager_graph(ops):
    """The captured call is refused before it launches anything; without the eager graph it runs."""
    order = ops.sort_tokens(choices(96, 4, 2, 3), 3)
    x, wt, d = rnd(97, 4, 16).requires_grad_(), rnd(98, 4, 2).requires_grad_(), rnd(99, 4, 16)
    f = lambda: ops.combine_tokens(ops.dispatch_tokens(x * 2.0, order), order, wt)  # x reaches it through another node
    alive = f()
    want = torch.autograd.grad(f(), (x, wt), d)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                f()
    torch.cuda.synchronize()
    del alive
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(f(), (x, wt), d)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_differentiable_once(ops):
    order = ops.sort_tokens(choices(110, 4, 2, 3), 3)
    x, wt = rnd(111, 4, 16).requires_grad_(), rnd(112, 4, 2).requires_grad_()
    y = ops.combine_tokens(ops.dispatch_tokens(x, order), order, wt)
    with pytest.raises(NotImplementedError, match="once"):
        torch.autograd.grad(y.sum(), (x, wt), create_graph=True)
    with torch.no_grad():
        assert not ops.combine_tokens(ops.dispatch_tokens(x, order), order, wt).requires_grad


def test_int8_experts_layer(ops):
    """Norm, route, sort, products, activation, products, combine: against 64 bits on the same codes.

    The steps round three times before the sum: gu to bf16 (2^-8), h to its code (half a scale step), ys to
    bf16; a change of g or u moves h by at most 1.1 |u| or |silu(g)| times it."""
    H, I, E, P, k = 512, 256, 16, 50, 4
    gen = torch.Generator().manual_seed(98)
    moe = ops.MoE(H, I, E, k, "fp8", layouts=("frag",))
    moe.load_router(ops.make_router(E, H, gen))
    ex = ops.Int8Experts(H, I, E)
    for e in range(E):
        ex.load_expert(e, ops.make_expert("fp8" if e % 2 else "fp4", H, I, gen))
    x, r, w = rnd(99, P, H, dtype=torch.bfloat16), rnd(100, P, H, dtype=torch.bfloat16), 1 + 0.1 * rnd(101, H)
    n = ops.rms_norm_quant(x, w, r, fmt="int8", normed=True)
    wt, idx = ops.Gate(moe)(n.normed)
    idx[3, 1] = -1
    idx[7] = -1
    y = ex(n.q, n.s, idx, wt)
    a = n.q.double() * n.s.double()[:, None]
    want, tol = torch.zeros(P, H, dtype=torch.float64, device="cuda"), torch.zeros(P, H, dtype=torch.float64, device="cuda")
    for t in range(P):
        for j in range(k):
            e = int(idx[t, j])
            if e < 0:
                continue
            gu = (ex.w13[e].double() @ a[t]) * ex.s13[e].double()
            g, u = gu[:I].clamp(max=10.0), gu[I:].clamp(-10.0, 10.0)
            h = g * torch.sigmoid(g) * u
            dh = 2.0 ** -8 * 1.01 * (1.1 * u.abs() * g.abs() + (g * torch.sigmoid(g)).abs() * u.abs())
            dh = dh + (h.abs() + dh).max() / 127 * 0.5 * 1.01
            w2, wj = ex.w2[e].double() * ex.s2[e].double()[:, None], abs(float(wt[t, j]))
            out = w2 @ h
            want[t] += float(wt[t, j]) * out
            step = w2.abs() @ dh
            tol[t] += wj * (step + 2.0 ** -8 * 1.01 * (out.abs() + step))
    within(y, want, (tol + 2.0 ** -8 * (want.abs() + tol)) * 1.001)
    assert not y[7].any()
    # beside the layer's own float formulas: int8 with one scale per row keeps the direction
    ref = torch.nn.functional.cosine_similarity(y.double(), want, dim=1)
    assert float(ref[torch.arange(P, device="cuda") != 7].min()) > 0.99


@pytest.mark.parametrize("rows,n", [(4096, 512), (3, 5120), (65, 16384)])
def test_scales_are_act_quants(ops, rows, n):
    """The same rows, in fp32, through act_quant and through a division per row: the same scales, to the last bit."""
    import kernel
    x, w = rnd(130, rows, n, scale=3.0), 1 + 0.2 * rnd(131, n)
    for scale_fmt in (None, "ue8m0"):
        got = ops.rms_norm_quant(x, w, normed=True, scale_fmt=scale_fmt)
        q, s = kernel.act_quant(got.normed, 128, scale_fmt)
        assert torch.equal(got.s, s)
        # codes: v times a reciprocal, within 8 u of the quotient: only values that near to a tie change sides. Ties lie
        # at least 2^-4 of the value apart, so these are 16 u / 2^-4 = 2^-16 of all values (twice that, and a few)
        other = q.view(torch.uint8) != got.q.view(torch.uint8)
        assert int(other.sum()) <= 8 + 2.0 ** -15 * other.numel()
    got = ops.rms_norm_quant(x, w, normed=True, fmt="int8")
    top = got.normed.abs().amax(-1).clamp(min=1e-4)
    assert torch.equal(got.s, torch.div(top, torch.full_like(top, 127.0)))


FAR = [-87.25, -88.0, -89.0, -104.0, -1e4, -1e30, -1e32, -1e36]


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt,n", [("fp8", 256), ("int8", 256), ("int8", 257), ("int8", 1500), ("int8", 1501)])
def test_swiglu_far_negative_gates(ops, fmt, n, dtype, weighted):
    """Gates down to the type's lowest value (a masked channel) are 0, and leave their row's scale alone."""
    far = FAR + [float(torch.finfo(dtype).min)]
    gu = rnd(140, 3 * len(far), 2 * n, dtype=dtype)
    gu[:, n:][:, ::7] = -10.0
    wr = rnd(141, gu.shape[0]) * 40.0 if weighted else None
    for i, g in enumerate(far):
        gu[3 * i, 5] = g        # one channel among others
        gu[3 * i + 1, :n] = g   # the whole row
        gu[3 * i + 2, :n:3] = g
    q, s = ops.swiglu_quant(gu, wr, fmt=fmt)
    v = swiglu_ref(gu, wr)
    # 17 roundings of the value; where the reciprocal of 1 + exp(-g) falls below fp32's normal range it is 0: 1e-36 u wr
    check_quant(q, s, v, fmt, 17 * U)
    assert not q[1::3].float().any() and bool((s[1::3] == torch.tensor(1e-4) / (448.0 if fmt == "fp8" else 127.0)).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt,n", [("fp8", 128), ("int8", 128), ("int8", 129)])
def test_swiglu_without_a_limit(ops, fmt, n, dtype):
    gu = rnd(142, 4, 2 * n, dtype=dtype, scale=20.0)
    top = float(torch.finfo(dtype).max)
    gu[1, 3], gu[1, n + 3] = top, 0.25
    gu[2, 3], gu[2, n + 3] = -top, top
    gu[3, 3], gu[3, n + 3] = 2.0 ** 100, 2.0 ** 20
    for limit in (float("inf"), top):
        q, s = ops.swiglu_quant(gu, limit=limit, fmt=fmt)
        check_quant(q, s, swiglu_ref(gu, None, limit), fmt, 16 * U)


@pytest.fixture
def operands_late():
    """Int8 products whose operands count as late from the first on."""
    from dsmoe import _lib as L
    L.call("dsmoe_int8_operand_wait", 0)
    yield
    L.call("dsmoe_int8_operand_wait", 1000000000)


# one-tile CTAs alone and in clusters of 2 to 8; pairs with fewer K blocks than ring stages, with more, several tiles each
@pytest.mark.parametrize("m,n,k", [(1, 128, 128), (8, 4096, 5120), (33, 64, 4096), (256, 1024, 2048), (4096, 512, 512),
                                   (1024, 4096, 5120), (4096, 4096, 5120)])
def test_int8_gemm_gives_nan_where_operands_are_late(ops, operands_late, m, n, k):
    from dsmoe import _lib as L
    a, b, sa, sb = codes(150, m, k), codes(151, n, k), scales(152, m), scales(153, n)
    got = ops.int8_gemm(a, sa, b, sb, out_dtype=torch.float32)
    torch.cuda.synchronize()
    L.call("dsmoe_int8_operand_wait", 1000000000)
    want = ops.int8_gemm(a, sa, b, sb, out_dtype=torch.float32)
    within(want, (a.double() @ b.double().T) * sa.double()[:, None] * sb.double(), product_tol(want.double(), torch.float32))
    assert bool(torch.isnan(got).all())  # both CTAs of a pair: neither stores the incomplete sums of the other's products


def test_int8_grouped_gemm_gives_nan_where_operands_are_late(ops, operands_late):
    from dsmoe import _lib as L
    for counts, n, k in (([1] * 6, 256, 512), ([700, 0, 900, 1500], 512, 2048)):
        m, e = sum(counts), len(counts)
        a, b, sa, sb = codes(154, m, k), codes(155, e, n, k), scales(156, m), scales(157, e, n)
        L.call("dsmoe_int8_operand_wait", 0)
        got = ops.int8_grouped_gemm(a, sa, b, sb, group_offsets(counts), out_dtype=torch.float32)
        torch.cuda.synchronize()
        L.call("dsmoe_int8_operand_wait", 1000000000)
        want = ops.int8_grouped_gemm(a, sa, b, sb, group_offsets(counts), out_dtype=torch.float32)
        assert bool(torch.isnan(got).all()) and not bool(torch.isnan(want).any())


@pytest.mark.parametrize("dtype", [torch.complex64, torch.complex128])
def test_dispatch_of_conjugates(ops, dtype):
    g = torch.Generator().manual_seed(160)
    z = torch.randn((5, 24), generator=g, dtype=dtype).to("cuda")
    order = ops.sort_tokens(torch.tensor([[1, 0], [2, -1], [0, 1], [1, 2], [0, 2]], device="cuda"), 3)
    for x in (z.conj(), z.conj()[:, 1:], z.conj().imag, z):
        want = torch.zeros((10, x.shape[1]), dtype=x.dtype, device="cuda")
        for t in range(5):
            for j in range(2):
                if order.pos[t, j] >= 0:
                    want[order.pos[t, j]] = x[t].resolve_conj()
        got = ops.dispatch_tokens(x, order)
        assert not got.is_conj() and not got.is_neg() and torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_negative_views(ops, dtype):
    """Views that are negated when they are read: as inputs like any other tensor, refused where a kernel would write them."""
    neg = torch._neg_view
    x, r, w, gu = rnd(161, 6, 256, dtype=dtype), rnd(162, 6, 256, dtype=dtype), rnd(163, 256), rnd(164, 6, 512, dtype=dtype)
    wr, flat = rnd(165, 6), torch.cat([x.new_zeros(1), x.flatten()])[1:].view(6, 256)
    bits = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
    same = lambda a, b: all((p is None and q is None) or torch.equal(bits(p), bits(q)) for p, q in zip(a, b))
    for fmt in ("fp8", "int8"):
        assert same(ops.rms_norm_quant(neg(x), neg(w), neg(r), fmt=fmt), ops.rms_norm_quant(-x, -w, -r, fmt=fmt))
        assert same(ops.rms_norm_quant(neg(flat), w, fmt=fmt), ops.rms_norm_quant(-x, w, fmt=fmt))
        assert same(ops.swiglu_quant(neg(gu), neg(wr), fmt=fmt), ops.swiglu_quant(-gu, -wr, fmt=fmt))
    a, b, sa, sb = codes(166, 6, 256), codes(167, 2, 512, 256), scales(168, 6), scales(169, 2, 512)
    off = group_offsets([2, 4])
    assert torch.equal(ops.int8_gemm(a, neg(sa), b[0], neg(sb[0])), ops.int8_gemm(a, sa, b[0], sb[0]))
    assert torch.equal(ops.int8_grouped_gemm(a, neg(sa), b, sb, off), ops.int8_grouped_gemm(a, -sa, b, sb, off))
    idx = torch.tensor([[0, 1], [2, -1], [1, 0]], device="cuda")
    assert same(ops.sort_tokens(neg(-idx), 3), ops.sort_tokens(idx, 3))
    order, wt = ops.sort_tokens(idx, 3), rnd(170, 3, 2)
    leaves = [t.clone().requires_grad_() for t in (x, wt)]
    y, want = ops.combine_tokens(neg(leaves[0]), order, neg(leaves[1])), ops.combine_tokens(-x, order, -wt)
    assert torch.equal(y, want)
    dy = rnd(171, 3, 256, dtype=dtype)
    got = torch.autograd.grad(y, leaves, neg(dy))
    leaves = [t.clone().requires_grad_() for t in (x, wt)]
    assert same(got, torch.autograd.grad(ops.combine_tokens(-leaves[0], order, -leaves[1]), leaves, -dy))
    for call in (lambda: ops.rms_norm_quant(x, w, neg(r), inplace=True),
                 lambda: ops.int8_gemm(a, sa, b[0], sb[0], out=neg(torch.zeros(6, 512, device="cuda", dtype=dtype))),
                 lambda: ops.combine_tokens(x, order._replace(pos=neg(order.pos)))):
        with pytest.raises(ValueError, match="negative view|must come from sort_tokens"):
            call()


def test_tensors_with_a_tangent_are_refused(ops):
    from torch.autograd import forward_ad as fwd
    x, w = torch.ones(2, 128).to("cuda"), torch.ones(128).to("cuda")
    q, s = torch.ones(2, 128, dtype=torch.int8).to("cuda"), torch.ones(2).to("cuda")
    order = ops.TokenOrder(torch.tensor([[0], [1]], dtype=torch.int32).to("cuda"), torch.tensor([0, 1], dtype=torch.int32).to("cuda"),
                           torch.tensor([0, 1, 2], dtype=torch.int32).to("cuda"))
    with fwd.dual_level():
        d = lambda t: fwd.make_dual(t, torch.ones_like(t))
        for call in (lambda: ops.rms_norm_quant(d(x), w), lambda: ops.rms_norm_quant(x, d(w)),
                     lambda: ops.rms_norm_quant(x, w, d(x)), lambda: ops.swiglu_quant(d(x)), lambda: ops.swiglu_quant(x, d(s)),
                     lambda: ops.int8_gemm(q, d(s), q, s), lambda: ops.int8_gemm(q, s, q, d(s)),
                     lambda: ops.int8_grouped_gemm(q, d(s), q[None], s[None], order.offsets[:2]),
                     lambda: ops.dispatch_tokens(d(x), order), lambda: ops.dispatch_tokens(x, order, d(s)),
                     lambda: ops.dispatch_tokens(d(x.clone().requires_grad_()), order),
                     lambda: ops.combine_tokens(d(x), order), lambda: ops.combine_tokens(x, order, d(s[:, None]))):
            with pytest.raises(ValueError, match="no forward-mode derivative"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="no forward-mode derivative"):
                call()
        assert torch.equal(ops.dispatch_tokens(fwd.unpack_dual(d(x)).primal, order), x)


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
def test_int8_experts_take_the_formats_types(ops, fmt):
    """Codes and scales as raw bytes or in their own types, from the CPU or the GPU: the same weights."""
    h, i = 288, 160
    ew = ops.make_expert(fmt, h, i, torch.Generator().manual_seed(1))
    typed = {n: t.view(torch.float8_e4m3fn) if fmt == "fp8" and n[0] == "w" else
             t.view(torch.float8_e8m0fnu) if fmt == "fp4" and n[0] == "s" else t for n, t in vars(ew).items() if n != "fmt"}
    layer = ops.Int8Experts(h, i, 3)
    for e, w in enumerate((ew, ops.ExpertWeights(fmt, **typed), ew.to("cuda"))):
        layer.load_expert(e, w)
    for t in (layer.w13, layer.s13, layer.w2, layer.s2):
        assert bool(t[0].any()) and torch.equal(t[0], t[1]) and torch.equal(t[0], t[2])


def test_int8_experts_take_packed_e2m1_in_its_own_type(ops):
    h, i = 288, 160
    ew = ops.make_expert("fp4", h, i, torch.Generator().manual_seed(2))
    own = {n: t.view(torch.float4_e2m1fn_x2) if n[0] == "w" else t for n, t in vars(ew).items() if n != "fmt"}
    layer = ops.Int8Experts(h, i, 2)
    layer.load_expert(0, ew)
    layer.load_expert(1, ops.ExpertWeights("fp4", **own))
    for t in (layer.w13, layer.s13, layer.w2, layer.s2):
        assert bool(t[0].any()) and torch.equal(t[0], t[1])
