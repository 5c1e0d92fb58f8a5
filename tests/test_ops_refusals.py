"""The 8-bit operators' C entry points refuse bad calls before they touch the device (no GPU here), and
their Python surface takes CUDA tensors only."""
import pytest
import torch

A = 4096  # an aligned address that no call may reach


def _code(name, *args):
    from dsmoe import _lib as L
    return getattr(L.lib, name)(*args)


NORM = dict(x=A, dtype=1, residual=2 * A, weight=3 * A, w_dtype=0, rows=4, hidden=256, eps=1e-6, q_dtype=2, pow2=0, q=A * 4,
            s=A * 8, residual_out=A * 12, normed=None, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(x=None), -1), (dict(weight=None), -1), (dict(q=None), -1), (dict(s=None), -1), (dict(dtype=2), -1),
    (dict(w_dtype=3), -1), (dict(q_dtype=1), -1), (dict(rows=0), -1), (dict(rows=-1), -1), (dict(rows=1 << 31), -1),
    (dict(hidden=0), -1), (dict(hidden=130), -1), (dict(hidden=16512), -1), (dict(residual=None), -1),
    (dict(q_dtype=3, pow2=1), -1), (dict(x=A + 2), -2), (dict(x=A + 1, q_dtype=3), -2), (dict(s=A * 8 + 2), -2),
    (dict(weight=3 * A + 2), -2), (dict(residual_out=2 * A + 64), -1), (dict(normed=A), -1), (dict(normed=A * 12), -1),
    (dict(q=A), -1), (dict(normed=2 * A + 512), -1)])
def test_rms_norm_quant_refuses(change, code):
    assert _code("dsmoe_rms_norm_quant", *{**NORM, **change}.values()) == code


SWIGLU = dict(gu=A, dtype=1, row_weight=None, rows=4, inter=256, limit=10.0, q_dtype=2, pow2=0, q=A * 4, s=A * 8, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(gu=None), -1), (dict(q=None), -1), (dict(s=None), -1), (dict(dtype=3), -1), (dict(q_dtype=0), -1), (dict(rows=0), -1),
    (dict(inter=100), -1), (dict(inter=0), -1), (dict(inter=16512), -1), (dict(limit=0.0), -1),
    (dict(limit=float("nan")), -1), (dict(q_dtype=3, pow2=1), -1), (dict(gu=A + 8), -2), (dict(gu=A + 1, q_dtype=3), -2),
    (dict(row_weight=A * 16 + 2), -2), (dict(q=A + 4000), -1)])
def test_swiglu_quant_refuses(change, code):
    assert _code("dsmoe_swiglu_quant", *{**SWIGLU, **change}.values()) == code


GEMM = dict(a=A, a_s=2 * A, M=4, K=64, b=3 * A, b_s=4 * A, N=32, out=5 * A, out_dtype=1, stream=None)
GROUPED = dict(a=A, a_s=2 * A, M=4, K=64, b=3 * A, b_s=4 * A, n_experts=3, N=32, offsets=6 * A, out=5 * A, out_dtype=1, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(a=None), -1), (dict(a_s=None), -1), (dict(b=None), -1), (dict(b_s=None), -1), (dict(out=None), -1), (dict(M=0), -1),
    (dict(N=0), -1), (dict(K=0), -1), (dict(K=24), -1), (dict(K=131072), -1), (dict(M=1 << 31), -1), (dict(N=1 << 31), -1),
    (dict(out_dtype=2), -1), (dict(a=A + 8), -2), (dict(b=A + 8), -2), (dict(a_s=2 * A + 1), -2), (dict(out=5 * A + 1), -2)])
def test_int8_gemm_refuses(change, code):
    assert _code("dsmoe_int8_gemm", *{**GEMM, **change}.values()) == code
    assert _code("dsmoe_int8_grouped_gemm", *{**GROUPED, **change}.values()) == code


@pytest.mark.parametrize("change,code", [(dict(offsets=None), -1), (dict(n_experts=0), -1), (dict(n_experts=1025), -1),
                                         (dict(offsets=6 * A + 2), -2), (dict(n_experts=1024, N=1 << 21), -1)])
def test_int8_grouped_gemm_refuses(change, code):
    assert _code("dsmoe_int8_grouped_gemm", *{**GROUPED, **change}.values()) == code


def test_token_entry_points_refuse():
    sort = dict(idx=A, P=4, k=2, n_experts=8, pos=2 * A, src=3 * A, offsets=4 * A, stream=None)
    for change, code in [(dict(idx=None), -1), (dict(pos=None), -1), (dict(src=None), -1), (dict(offsets=None), -1),
                         (dict(P=0), -1), (dict(k=0), -1), (dict(k=65), -1), (dict(n_experts=0), -1), (dict(n_experts=1025), -1),
                         (dict(P=1 << 30), -1), (dict(P=1 << 40, k=64), -1), (dict(idx=A + 4), -2), (dict(pos=A + 2), -2)]:
        assert _code("dsmoe_sort_tokens", *{**sort, **change}.values()) == code, change
    disp = dict(x=A, s=None, pos=2 * A, offsets=3 * A, n_experts=8, P=4, k=2, row_bytes=64, xs=4 * A, ss=None, stream=None)
    for change, code in [(dict(x=None), -1), (dict(xs=None), -1), (dict(pos=None), -1), (dict(offsets=None), -1),
                         (dict(s=A), -1), (dict(ss=A), -1), (dict(row_bytes=0), -1), (dict(row_bytes=1 << 31), -1),
                         (dict(pos=2 * A + 1), -2)]:
        assert _code("dsmoe_dispatch_rows", *{**disp, **change}.values()) == code, change
    comb = dict(ys=A, dtype=1, pos=2 * A, wt=None, P=4, k=2, width=64, y=3 * A, stream=None)
    for change, code in [(dict(ys=None), -1), (dict(y=None), -1), (dict(pos=None), -1), (dict(dtype=2), -1), (dict(width=0), -1),
                         (dict(width=1 << 29), -1), (dict(ys=A + 1), -2), (dict(wt=A + 1), -2)]:
        assert _code("dsmoe_combine_rows", *{**comb, **change}.values()) == code, change
    grad = dict(dy=A, ys=2 * A, dtype=1, pos=3 * A, wt=4 * A, offsets=5 * A, n_experts=8, P=4, k=2, width=64, dys=6 * A,
                dwt=7 * A, stream=None)
    for change, code in [(dict(dy=None), -1), (dict(ys=None), -1), (dict(pos=None), -1), (dict(offsets=None), -1),
                         (dict(dys=None, dwt=None), -1), (dict(dtype=3), -1), (dict(width=0), -1), (dict(dys=A + 1), -2),
                         (dict(dwt=A + 2), -2)]:
        assert _code("dsmoe_combine_grad", *{**grad, **change}.values()) == code, change


def test_outputs_are_their_own_memory():
    """One byte in common is enough, whichever end; neighbours are fine as far as this check goes."""
    norm, gemm = {**NORM, "residual_out": 2 * A}, {**GROUPED, "out": 5 * A}
    for name, args, change in (
            ("dsmoe_rms_norm_quant", norm, dict(weight=2 * A + 2032)), ("dsmoe_rms_norm_quant", norm, dict(s=3 * A + 1020)),
            ("dsmoe_rms_norm_quant", norm, dict(s=A - 28)), ("dsmoe_rms_norm_quant", norm, dict(s=4 * A)),
            ("dsmoe_swiglu_quant", SWIGLU, dict(row_weight=8 * A + 28)), ("dsmoe_swiglu_quant", SWIGLU, dict(s=A + 4092)),
            ("dsmoe_int8_gemm", GEMM, dict(out=A + 254)), ("dsmoe_int8_gemm", GEMM, dict(out=2 * A - 254)),
            ("dsmoe_int8_gemm", GEMM, dict(out=3 * A + 2046)), ("dsmoe_int8_gemm", GEMM, dict(out=4 * A + 126)),
            ("dsmoe_int8_grouped_gemm", gemm, dict(out=3 * A + 6142)), ("dsmoe_int8_grouped_gemm", gemm, dict(out=6 * A + 14)),
            ("dsmoe_int8_grouped_gemm", gemm, dict(out=4 * A + 382))):
        assert _code(name, *{**args, **change}.values()) == -1, (name, change)
    sort = dict(idx=A, P=4, k=2, n_experts=8, pos=2 * A, src=3 * A, offsets=4 * A, stream=None)
    disp = dict(x=A, s=5 * A, pos=2 * A, offsets=3 * A, n_experts=8, P=4, k=2, row_bytes=64, xs=4 * A, ss=6 * A, stream=None)
    comb = dict(ys=A, dtype=1, pos=2 * A, wt=4 * A, P=4, k=2, width=64, y=3 * A, stream=None)
    grad = dict(dy=A, ys=2 * A, dtype=1, pos=3 * A, wt=4 * A, offsets=5 * A, n_experts=8, P=4, k=2, width=64, dys=6 * A,
                dwt=7 * A, stream=None)
    for name, args, change in (
            ("dsmoe_sort_tokens", sort, dict(pos=A + 60)), ("dsmoe_sort_tokens", sort, dict(src=2 * A + 28)),
            ("dsmoe_sort_tokens", sort, dict(offsets=A - 32)), ("dsmoe_dispatch_rows", disp, dict(xs=A + 240)),
            ("dsmoe_dispatch_rows", disp, dict(ss=4 * A + 508)), ("dsmoe_dispatch_rows", disp, dict(ss=5 * A + 12)),
            ("dsmoe_combine_rows", comb, dict(y=A + 1008)), ("dsmoe_combine_rows", comb, dict(y=4 * A + 28)),
            ("dsmoe_combine_grad", grad, dict(dys=A + 496)), ("dsmoe_combine_grad", grad, dict(dys=2 * A - 1008)),
            ("dsmoe_combine_grad", grad, dict(dwt=6 * A + 1020)), ("dsmoe_combine_grad", grad, dict(dwt=5 * A + 32))):
        assert _code(name, *{**args, **change}.values()) == -1, (name, change)


def test_python_surface_takes_cuda_tensors_only():
    import dsmoe
    x, w = torch.zeros(2, 128), torch.ones(128)
    q, s, g = torch.zeros(2, 128, dtype=torch.int8), torch.ones(2), torch.zeros(2, 128, requires_grad=True)
    order = dsmoe.TokenOrder(torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                             torch.zeros(3, dtype=torch.int32))
    for call in (lambda: dsmoe.rms_norm_quant(x, w), lambda: dsmoe.swiglu_quant(x), lambda: dsmoe.int8_gemm(q, s, q, s),
                 lambda: dsmoe.int8_grouped_gemm(q, s, q[None], s[None], order.offsets),
                 lambda: dsmoe.sort_tokens(torch.zeros(2, 1, dtype=torch.int64), 2),
                 lambda: dsmoe.dispatch_tokens(x, order), lambda: dsmoe.combine_tokens(x, order),
                 lambda: dsmoe.dispatch_tokens(g, order), lambda: dsmoe.combine_tokens(g, order)):
        with pytest.raises(ValueError, match=r"CUDA tensors only, got \[2, .*\] on cpu"):
            call()


def test_native_half_refuses_other_objects():
    import dsmoe
    from dsmoe import _ops
    for call in (lambda: dsmoe.swiglu_quant(3), lambda: dsmoe.int8_gemm(None, None, None, None),
                 lambda: dsmoe.rms_norm_quant(torch.ones(2), [1.0]), lambda: dsmoe.sort_tokens(torch.zeros(2, 1), None),
                 lambda: dsmoe.int8_grouped_gemm(1, 2, 3, 4, None), lambda: _ops.combine_tokens(1, 2)):
        with pytest.raises(TypeError):
            call()


def test_kernel_surface_offers_the_operators():
    import dsmoe
    import kernel
    assert kernel.int8_gemm is dsmoe.int8_gemm and kernel.rms_norm_quant is dsmoe.rms_norm_quant
    assert kernel.swiglu_quant is dsmoe.swiglu_quant


def test_quant_int8_channel():
    from dsmoe.synth import quant_int8_channel
    w = torch.randn((7, 33), generator=torch.Generator().manual_seed(0))
    w[3] = 0.0
    q, s = quant_int8_channel(w)
    assert q.dtype == torch.int8 and s.shape == (7,) and int(q.abs().max()) == 127 and not q[3].any()
    assert bool(((q.double() * s.double()[:, None] - w.double()).abs() <= s.double()[:, None] * (0.5 + 127 * 2.0 ** -22)).all())


def test_int8_operand_wait_refuses():
    assert _code("dsmoe_int8_operand_wait", -1) == -1 and _code("dsmoe_int8_operand_wait", 1000000001) == -1
    assert _code("dsmoe_int8_operand_wait", 1000000000) == 0


def test_tensors_with_a_tangent_are_refused():
    import dsmoe as ops
    from torch.autograd import forward_ad as fwd
    x, w = torch.ones(2, 128), torch.ones(128)
    q, s = torch.ones(2, 128, dtype=torch.int8), torch.ones(2)
    order = ops.TokenOrder(torch.tensor([[0], [1]], dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32),
                           torch.tensor([0, 1, 2], dtype=torch.int32))
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


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
def test_int8_experts_refuse_weights_that_are_not_there(fmt):
    """Codes and scales whose shape or type is not the format's never reach a kernel (none runs here: no GPU is needed)."""
    import dsmoe
    h, i = 288, 160
    ew = dsmoe.make_expert(fmt, h, i, torch.Generator().manual_seed(0))
    layer = dsmoe.Int8Experts(h, i, 2, device="cpu")
    layer.w13.fill_(1)
    short = {"s1": ew.s1[:-1], "s3": ew.s3[:, :-1], "s2": ew.s2.flatten(), "w1": ew.w1[:-1], "w2": ew.w2[:, :-16], "w3": ew.w3[None]}
    wrong = {"s1": ew.s1.to(torch.float64), "s3": ew.s3.to(torch.bfloat16), "s2": ew.s2.to(torch.int32), "w1": ew.w1.to(torch.int16),
             "w2": ew.w2.float()}
    wrong["s3"] = ew.s3.to(torch.uint8) if fmt == "fp8" else ew.s3.float()  # the other format's type
    for error, changes in ((ValueError, short), (TypeError, wrong)):
        for name, value in changes.items():
            with pytest.raises(error, match="codes"):
                layer.load_expert(0, dsmoe.ExpertWeights(**{**vars(ew), name: value}))
    with pytest.raises(ValueError, match="expert format"):
        layer.load_expert(0, dsmoe.ExpertWeights(**{**vars(ew), "fmt": "int4"}))
    with pytest.raises(IndexError):
        layer.load_expert(2, ew)
    if fmt == "fp4":  # hidden and inter in steps of 16 are the layer's; FP4 comes in groups of 32
        odd = dsmoe.Int8Experts(304, i, 1, device="cpu")
        with pytest.raises(ValueError, match="multiple of 32"):
            odd.load_expert(0, ew)
    assert bool((layer.w13 == 1).all())
