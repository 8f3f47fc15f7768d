"""Host side of the feed-forward layer's calls: what they refuse, with the status and before anything runs, and the
scratch that they ask for.  No GPU needed."""
import ctypes

import pytest

import t0g

A, B, C, D, E, F, G, H = (0x10000000 * i for i in range(1, 9))


def norm(**kw):
    return _with(t0g.rms_norm_desc(A, B, 16, 300, residual=C, sum=D, y=E, q=F, scales=G), kw)


def norm_backward(**kw):
    return _with(t0g.rms_norm_backward_desc(A, B, C, 16, 300, dsum=D, dx=E, dw=F), kw)


def quantize(**kw):
    return _with(t0g.fp8_quantize_desc(A, B, C, 16, 300, qt=D, scales_t=E), kw)


def gemm(**kw):
    return _with(t0g.fp8_gemm_desc(A, B, C, D, E, 16, 256, 300), kw)


def gated(**kw):
    return _with(t0g.gated_linear_desc(A, B, C, D, 16, 256, 72, gate=E, up=F), kw)


def gated_backward(**kw):
    return _with(t0g.gated_linear_backward_desc(A, B, C, D, 16, 256, 72, gate=E, up=F, dx=G, dwg=H, dwu=2 * H), kw)


def _with(d, kw):
    for k, v in kw.items():
        assert hasattr(d, k), k
        setattr(d, k, v)
    return d


CALLS = {t0g.RmsNormDesc: "rms_norm", t0g.RmsNormBackwardDesc: "rms_norm_backward", t0g.Fp8QuantizeDesc: "fp8_quantize",
         t0g.Fp8GemmDesc: "fp8_gemm", t0g.GatedLinearDesc: "gated_linear", t0g.GatedLinearBackwardDesc: "gated_linear_backward"}


def call(d):
    """On no device: the descriptor is checked first."""
    t0g.GpuRuntime.__dict__[CALLS[type(d)]](t0g.GpuRuntime(None), d)


def refused(d, word):
    for f in [call] + ([t0g.ffn_scratch_size] if type(d) in t0g._FFN_SCRATCH else []):
        with pytest.raises(t0g.T0gError) as e:
            f(d)
        assert e.value.code == t0g.ERR_INVALID_ARG
        assert word in str(e.value), str(e.value)


@pytest.mark.parametrize("make", [norm, norm_backward, quantize, gemm, gated, gated_backward])
def test_a_good_descriptor_needs_a_device(make):
    with pytest.raises(t0g.T0gError) as e:
        call(make())
    assert e.value.code == t0g.ERR_INVALID_ARG and "device is NULL" in str(e.value)


@pytest.mark.parametrize("name", sorted(CALLS.values()))
def test_null_descriptor(name):
    assert getattr(t0g._lib, "t0g_" + name)(None, None) == t0g.ERR_INVALID_ARG
    if name in t0g._FFN_SCRATCH.values():
        n = ctypes.c_size_t()
        assert getattr(t0g._lib, f"t0g_{name}_scratch_size")(None, ctypes.byref(n)) == t0g.ERR_INVALID_ARG


@pytest.mark.parametrize("change,word", [
    ({"hidden": 0}, "size"), ({"hidden": t0g.NORM_MAX + 1}, "size"), ({"rows": 1 << 31}, "size"), ({"eps": -1.0}, "eps"),
    ({"eps": float("nan")}, "eps"), ({"weight_offset": float("inf")}, "weight_offset"), ({"x_dtype": 2}, "x_dtype"),
    ({"residual_dtype": 3}, "residual_dtype"), ({"weight_dtype": 2}, "weight_dtype"), ({"sum_dtype": 4}, "sum_dtype"),
    ({"y_dtype": t0g.E4M3}, "y_dtype"), ({"q_dtype": t0g.BF16}, "q_dtype"), ({"q_dtype": 4}, "q_dtype"), ({"x": 0}, "NULL"),
    ({"sum": 0, "y": 0, "q": 0, "scales": 0}, "output"), ({"q": 0}, "together"), ({"scales": 0}, "together"),
    ({"ldx": 299}, "x"), ({"ldr": 1}, "residual"), ({"ldsum": 299}, "sum"), ({"ldy": 299}, "y"), ({"ldq": 299}, "q"), ({"ldsc": 15}, "scales"),
    ({"x": A + 1}, "aligned"), ({"weight": B + 1}, "aligned"), ({"scales": G + 2}, "aligned"), ({"y": E + 2, "y_dtype": 0}, "aligned"),
    ({"y": C}, "overlaps"), ({"sum": A + 2}, "overlaps"), ({"sum": A, "sum_dtype": 0}, "overlaps"), ({"sum": C, "ldsum": 301}, "overlaps"),
    ({"y": A + 16 * 600 - 2}, "overlaps"), ({"q": E}, "overlaps"), ({"q": A}, "overlaps"), ({"scales": F + 16}, "overlaps"), ({"y": B}, "overlaps"),
    ({"sum": A, "y": A}, "overlaps"),
])
def test_norm_refusals(change, word):
    refused(norm(**change), word)


@pytest.mark.parametrize("change", [{"sum": A}, {"sum": C}, {"y": A}, {"y": A + 16 * 600}, {"weight": 0}, {"residual": 0}, {"y": 0}, {"sum": 0},
                                    {"q": 0, "scales": 0}, {"ldsc": 40}, {"rows": 0, "x": 0}])
def test_norm_takes(change):
    with pytest.raises(t0g.T0gError, match="device is NULL"):
        call(norm(**change))


@pytest.mark.parametrize("change,word", [
    ({"hidden": 0}, "size"), ({"hidden": t0g.NORM_MAX + 1}, "size"), ({"eps": float("inf")}, "eps"), ({"dy_dtype": 2}, "dy_dtype"),
    ({"x_dtype": 2}, "x_dtype"), ({"weight_dtype": 2}, "weight_dtype"), ({"dsum_dtype": 2}, "dsum_dtype"), ({"dx_dtype": 2}, "dx_dtype"),
    ({"dw_dtype": 2}, "dw_dtype"), ({"dx": 0, "dw": 0}, "output"), ({"dy": 0}, "NULL"), ({"x": 0}, "NULL"), ({"lddy": 299}, "dy"),
    ({"ldds": 299}, "dsum"), ({"lddx": 299}, "dx"), ({"dw": F + 2}, "aligned"), ({"dx": C}, "overlaps"), ({"dw": A}, "overlaps"),
    ({"dx": A, "lddx": 304}, "overlaps"), ({"dx": B, "dx_dtype": 0}, "overlaps"), ({"dw": E}, "overlaps"),
])
def test_norm_backward_refusals(change, word):
    refused(norm_backward(**change), word)


def test_norm_backward_scratch():
    assert t0g.ffn_scratch_size(norm_backward(dw=0)) == 0
    assert t0g.ffn_scratch_size(norm_backward()) >= 304 * 4
    for a in (A, B, D):
        assert t0g.ffn_scratch_size(norm_backward(dx=a)) == t0g.ffn_scratch_size(norm_backward())


@pytest.mark.parametrize("change,word", [
    ({"cols": 0}, "size"), ({"cols": (1 << 30) + 1}, "size"), ({"rows": (1 << 30) + 1}, "size"), ({"x_dtype": 2}, "x_dtype"),
    ({"q_dtype": 1}, "q_dtype"), ({"block": 2}, "block"), ({"q": 0, "scales": 0, "qt": 0, "scales_t": 0}, "output"), ({"q": 0}, "together"),
    ({"scales_t": 0}, "together"), ({"x": 0}, "NULL"), ({"ldx": 299}, "x"), ({"ldq": 299}, "q"), ({"ldsc": 15}, "scales"),
    ({"ldqt": 15}, "qt"), ({"ldsct": 299}, "scales_t"), ({"x": A + 1}, "aligned"), ({"scales": C + 1}, "aligned"), ({"q": A}, "overlaps"),
    ({"qt": B + 4799}, "overlaps"), ({"scales_t": C}, "overlaps"), ({"block": 1, "ldsct": 2}, "scales_t"),
])
def test_quantize_refusals(change, word):
    refused(quantize(**change), word)


@pytest.mark.parametrize("change,word", [
    ({"k": 0}, "size"), ({"k": 1 << 23}, "size"), ({"m": (1 << 28) + 1}, "size"), ({"n": (1 << 26) + 1}, "size"), ({"a_dtype": 1}, "a_dtype"),
    ({"b_dtype": 0}, "b_dtype"), ({"out_dtype": 2}, "out_dtype"), ({"b_block": 2}, "b_block"), ({"a": 0}, "NULL"), ({"b": 0}, "NULL"),
    ({"c": 0}, "NULL"), ({"a_scales": 0}, "NULL"), ({"b_scales": 0}, "NULL"), ({"lda": 299}, "a"), ({"ldb": 299}, "b"), ({"ldc": 255}, "c"),
    ({"ldas": 15}, "a_scales"), ({"ldbs": 1}, "b_scales"), ({"b_block": 0, "ldbs": 255}, "b_scales"), ({"c": E + 1}, "aligned"),
    ({"a_scales": B + 2}, "aligned"), ({"c": A}, "overlaps"), ({"c": D}, "overlaps"), ({"c": C + 1024}, "overlaps"),
])
def test_gemm_refusals(change, word):
    refused(gemm(**change), word)


def test_gemm_scratch_is_for_unaligned_operands():
    assert t0g.ffn_scratch_size(gemm(k=304)) == 0
    assert t0g.ffn_scratch_size(gemm(m=0, n=0)) == 0


@pytest.mark.parametrize("change,word", [
    ({"features": 0}, "size"), ({"hidden": 0}, "size"), ({"hidden": 1 << 22}, "size"), ({"rows": 1 << 31}, "size"), ({"transpose": t0g.TN}, "transpose"),
    ({"activation": 0}, "activation"), ({"activation": t0g.OP_ABS}, "activation"), ({"h_dtype": 2}, "h_dtype"), ({"x": 0}, "NULL"),
    ({"wg": 0}, "NULL"), ({"wu": 0}, "NULL"), ({"h": 0}, "NULL"), ({"ldx": 71}, "x"), ({"ldw": 71}, "wg"), ({"ldh": 255}, "h"),
    ({"ldg": 255}, "gate"), ({"transpose": t0g.NN, "ldw": 255}, "wg"), ({"x": A + 1}, "aligned"), ({"h": A}, "overlaps"), ({"h": B + 2}, "overlaps"),
    ({"gate": D}, "overlaps"), ({"up": E}, "overlaps"), ({"up": C}, "overlaps"),
])
def test_gated_refusals(change, word):
    refused(gated(**change), word)


@pytest.mark.parametrize("change,word", [
    ({"features": 0}, "size"), ({"hidden": 0}, "size"), ({"transpose": 3}, "transpose"), ({"activation": 99}, "activation"),
    ({"dh_dtype": 2}, "dh_dtype"), ({"dx_dtype": 2}, "dx_dtype"), ({"dw_dtype": 2}, "dw_dtype"), ({"reserved": 1}, "reserved"),
    ({"dx": 0, "dwg": 0, "dwu": 0}, "output"), ({"gate": 0}, "together"), ({"up": 0}, "together"), ({"dh": 0}, "NULL"), ({"x": 0}, "NULL"),
    ({"lddh": 255}, "dh"), ({"lddx": 71}, "dx"), ({"lddw": 71}, "dwg"), ({"dx": B}, "overlaps"), ({"dwg": C}, "overlaps"), ({"dwu": H}, "overlaps"),
    ({"dx": A}, "overlaps"), ({"dwu": E}, "overlaps"), ({"dx": G + 2, "dx_dtype": 0}, "aligned"),
])
def test_gated_backward_refusals(change, word):
    refused(gated_backward(**change), word)


def test_gated_takes_optional_arrays():
    for change in ({"gate": 0}, {"up": 0}, {"gate": 0, "up": 0}, {"wu": B}, {"rows": 0, "x": 0, "h": 0}):
        with pytest.raises(t0g.T0gError, match="device is NULL"):
            call(gated(**change))
    for change in ({"gate": 0, "up": 0}, {"dx": 0}, {"dwg": 0}, {"dwu": 0}, {"dx": 0, "dwu": 0}):
        assert t0g.ffn_scratch_size(gated_backward(**change)) > 0


def test_columns_of_one_tensor_do_not_overlap():
    """Both weights' gradients as columns of one, and an output between its input's rows."""
    nn = dict(transpose=t0g.NN, ldw=512, lddw=512, dwu=H + 512)
    assert t0g.ffn_scratch_size(gated_backward(**nn)) > 0
    refused(gated_backward(**{**nn, "dwu": H + 510}), "overlaps")
    refused(gated_backward(**{**nn, "lddw": 511}), "overlaps")
    with pytest.raises(t0g.T0gError, match="device is NULL"):
        call(norm(ldx=600, ldy=600, y=A + 600))
    refused(norm(ldx=600, ldy=600, y=A + 598), "overlaps")
    refused(norm(ldx=599, ldy=599, y=A + 600), "overlaps")
