"""StreamingLinear.product against its formula in 64 bits (operator_reference.py has the bounds)."""
import math

import pytest
import torch

import operator_reference as ref
from helpers import calibrated_weight, outlier_weight, packed_from_int8, int8_mix, student_t_weight

pytestmark = pytest.mark.gpu

PARTS = [(None, False, False), ("silu", True, False), ("none", False, True), ("gelu_tanh", True, True)]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


def _layer(dev, out_f, in_f, recipe="t", level_bits=(3, 5, 8), bias=False, lanes=True, seed=0):
    """A layer and its dequantised weight, on the GPU from the start where that is large."""
    from ixrun_amd import StreamingLinear
    from ixrun_amd.quantize import decode_to_weight, int8x_quantize, quantize_for_deploy

    if recipe == "mix8":  # most of the weights above 15: a plane of 8 bits
        packed = packed_from_int8(int8_mix("only_l3", out_f * in_f, seed), out_f, in_f, level_bits=level_bits)
    elif out_f * in_f > 1 << 22:
        g = torch.Generator(dev).manual_seed(seed)
        w = torch.randn(out_f, in_f, generator=g, device=dev) * 0.02
        w[0, 0] = {"t": 0.7, "real": 0.2}[recipe]
        packed = quantize_for_deploy(w.bfloat16(), level_bits)
    else:
        make = {"t": student_t_weight, "outlier": outlier_weight, "real": lambda o, i, seed: calibrated_weight(o, i, seed, scale=0.0123046875 / 8)[0]}[recipe]
        packed = int8x_quantize(make(out_f, in_f, seed=seed), level_bits)
    b = (torch.randn(out_f, generator=torch.Generator().manual_seed(seed)) * 0.5).bfloat16() if bias else None
    layer = StreamingLinear(packed, bias=b, lanes=lanes)
    if out_f * in_f > 1 << 22:
        flat = torch.empty(out_f * in_f, dtype=torch.bfloat16, device=dev)
        layer._dp.decode(*layer._decode_table(), out_bf16=flat)
        return layer, flat.view(out_f, in_f), b.to(dev) if bias else None
    return layer, decode_to_weight(packed).to(dev), b.to(dev) if bias else None


def _operands(dev, rows, out_f, in_f, multiplier, residual, seed=1):
    g = torch.Generator(dev).manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g, device=dev).bfloat16()
    return make(rows, in_f), make(rows, out_f) if multiplier else None, make(rows, out_f) if residual else None


def _close(y, want, bound):
    off = (y.double() - want).abs()
    assert y.dtype == torch.bfloat16 and y.shape == want.shape
    assert bool((off <= bound).all()), f"{int((off > bound).sum())} of {off.numel()} elements, worst {float((off / bound).max()):.2f} bounds"


def _check(dev, layer, w, bias, rows, act, multiplier, residual, apart=False, seed=1):
    x, m, r = _operands(dev, rows, *w.shape, multiplier, residual, seed)
    _close(layer.product(x, act, m, r), *ref.epilogue(x, w, bias, act, m, r, apart=apart))


@pytest.mark.parametrize("recipe,level_bits", [("t", (3, 5, 8)), ("outlier", (4, 8)), ("real", (3, 5, 8)), ("mix8", (3, 5, 8))])
@pytest.mark.parametrize("out_f,in_f", [(256, 512), (640, 4608), (1001, 2056)])
@pytest.mark.parametrize("rows", [1, 2, 4, 7, 8, 13, 16, 17, 50, 100, 200])
def test_products_by_scheme_and_rows(dev, recipe, level_bits, out_f, in_f, rows):
    """Planes of 3, 4, 5 and 8 bits; every kind of epilogue once."""
    layer, w, bias = _layer(dev, out_f, in_f, recipe, level_bits, bias=rows % 2 == 0)
    act, multiplier, residual = PARTS[(rows + out_f) % 4]
    _check(dev, layer, w, bias, rows, act, multiplier, residual)


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh", "relu", "relu2"])
@pytest.mark.parametrize("rows", [1, 6, 40])
def test_products_by_activation(dev, act, rows):
    layer, w, bias = _layer(dev, 320, 1024, "outlier", bias=True)
    for multiplier in (False, True):
        for residual in (False, True):
            _check(dev, layer, w, bias, rows, act, multiplier, residual)


@pytest.mark.parametrize("out_f,in_f", [(1, 1), (3, 17), (5, 513), (64, 64), (33, 2047), (2000, 520)])
@pytest.mark.parametrize("rows", [1, 3, 16])
def test_products_of_odd_sizes(dev, out_f, in_f, rows):
    layer, w, bias = _layer(dev, out_f, in_f, "outlier", bias=True)
    _check(dev, layer, w, bias, rows, "silu", True, True, apart=layer._lanes is None)


@pytest.mark.parametrize("out_f,in_f,rows", [
    (17408, 5120, 1), (5120, 17408, 1), (5120, 17408, 12), (17408, 5120, 5), (40960, 2048, 3), (4096, 36864, 2), (5120, 17408, 300), (17408, 5120, 129),
    (32768, 1024, 400), (12288, 6144, 530), (2048, 2048, 700),
])
def test_large_products(dev, out_f, in_f, rows):
    """The kernels of large layers: sums by wave, several slices and one, whole tiles of a prompt and parts of them."""
    layer, w, bias = _layer(dev, out_f, in_f, "t", bias=True)
    _check(dev, layer, w, bias, rows, "gelu_tanh", True, True)


def test_a_long_prompt_is_taken_in_parts(dev):
    layer, w, bias = _layer(dev, 96, 256, "t", bias=True)
    _check(dev, layer, w, bias, 4096 + 31, "silu", True, True)


@pytest.mark.parametrize("rows", [1, 9, 33])
@pytest.mark.parametrize("how", ["no lanes", "odd rows", "fp32 bias"])
def test_products_whose_kernel_has_no_epilogue(dev, rows, how):
    layer, w, bias = _layer(dev, 72, 1023 if how == "odd rows" else 1024, "outlier", bias=True, lanes=how != "no lanes")
    layer._set_shared_buf(torch.empty(layer.N, dtype=torch.bfloat16, device=dev))
    if how == "fp32 bias":
        layer._bias = layer._bias.float()
        layer._bind()
    _check(dev, layer, w, bias, rows, "silu", True, True, apart=True)


def test_a_product_without_an_epilogue_is_the_forward(dev):
    layer, _, _ = _layer(dev, 640, 1536, "t")
    for rows in (1, 4, 12, 40):
        x = _operands(dev, rows, 640, 1536, False, False)[0]
        assert torch.equal(layer.product(x), layer(x))


def test_products_of_views(dev):
    layer, _, _ = _layer(dev, 200, 264, "t")
    for rows in (1, 6, 30):
        x, m, r = _operands(dev, rows, 200, 264, True, True)
        want = layer.product(x, "silu", m, r)
        wide = torch.full((rows, 500), math.nan, dtype=torch.bfloat16, device=dev)
        for start in (0, 1, 8):
            view = wide[:, start:start + 264]
            assert torch.equal(layer.product(view.copy_(x), "silu", m, r), want)
            view = wide[:, start:start + 200]
            assert torch.equal(layer.product(x, "silu", view.copy_(m), r), want)
            assert torch.equal(layer.product(x, "silu", m, view.copy_(r)), want)
        assert torch.equal(layer.product(x.t().contiguous().t(), "silu", m.t().contiguous().t(), r.t().contiguous().t()), want)
        deep = layer.product(x.view(1, rows, 264), "silu", m.view(1, rows, 200), r.view(1, rows, 200))
        assert deep.shape == (1, rows, 200) and torch.equal(deep[0], want)
    assert torch.equal(layer.product(x[0], "silu", m[0], r[0]), layer.product(x[:1], "silu", m[:1], r[:1])[0])
    assert layer.product(x[:0], "silu", m[:0], r[:0]).shape == (0, 200)


def test_infinities_and_nan_stay_in_their_rows(dev):
    layer, _, _ = _layer(dev, 128, 512, "t")
    for rows in (3, 12, 60):
        x, m, r = _operands(dev, rows, 128, 512, True, True)
        y = layer.product(x, "silu", m, r)
        x[1, 7], m[2, 5], r[2, 6] = math.nan, math.inf, -math.inf
        z = layer.product(x, "silu", m, r)
        assert bool(z[1].isnan().all()) and torch.equal(z[0], y[0]) and torch.equal(z[3:], y[3:])
        assert z[2, 6] == -math.inf and not bool(z[2, 5].isfinite()) and torch.equal(z[2, 7:], y[2, 7:])


def test_product_refusals(dev):
    layer, _, _ = _layer(dev, 64, 128)
    x, m, r = _operands(dev, 3, 64, 128, True, True)
    with pytest.raises(TypeError):
        layer.product(x.float())
    with pytest.raises(TypeError):
        layer.product(x, None, m.float())
    with pytest.raises(ValueError):
        layer.product(x[:, :100])
    with pytest.raises(ValueError):
        layer.product(x, None, m[:2])
    with pytest.raises(ValueError):
        layer.product(x, None, None, r[:, :5])
    with pytest.raises(ValueError, match="activation"):
        layer.product(x, "swish")
    with pytest.raises(RuntimeError):
        layer.product(x.cpu())
    with pytest.raises(RuntimeError, match="no gradient"):
        layer.product(x.clone().requires_grad_())


@pytest.mark.parametrize("rows", [1, 10, 70])
def test_a_gated_block_from_a_graph_and_another_stream(dev, rows):
    """Three products in a row, as a block makes them."""
    gate, w_gate, _ = _layer(dev, 768, 512, "t", seed=1)
    up, w_up, _ = _layer(dev, 768, 512, "t", seed=2)
    down, w_down, _ = _layer(dev, 512, 768, "t", seed=3)
    x = _operands(dev, rows, 1, 512, False, False)[0]

    def block(x):
        return down.product(gate.product(x, "silu", up(x)), residual=x)

    want = block(x)
    _close(up(x), *ref.epilogue(x, w_up))
    h = gate.product(x, "silu", up(x))
    _close(h, *ref.epilogue(x, w_gate, act="silu", multiplier=up(x)))
    _close(want, *ref.epilogue(h, w_down, residual=x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = block(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block(x)
    for seed in range(3):
        x.copy_(_operands(dev, rows, 1, 512, False, False, seed=seed + 10)[0])
        graph.replay()
        eager = block(x)
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


def test_a_layer_off_the_gpu_is_refused(dev):
    layer, _, _ = _layer(dev, 64, 128)
    x, m, r = _operands(dev, 3, 64, 128, True, True)
    want = layer.product(x, "silu", m, r)
    layer.cpu()
    for given in (x, x.cpu()):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            layer.product(given, "silu")
    layer.to(dev)
    assert torch.equal(layer.product(x, "silu", m, r), want)


@pytest.mark.parametrize("out_f,in_f", [(72, 1023), (100, 513), (33, 263), (640, 2049), (5126, 5003)])
@pytest.mark.parametrize("rows", [17, 40, 150, 520])
def test_prompts_of_odd_rows(dev, out_f, in_f, rows):
    """Rows that are no whole 16-byte pieces, one rounding all the same; views of them, and infinities next to what fills them up."""
    layer, w, bias = _layer(dev, out_f, in_f, "outlier" if out_f < 5000 else "t", bias=True)
    assert layer._lanes is not None
    _check(dev, layer, w, bias, rows, "gelu_tanh", True, True)
    x, m, r = _operands(dev, rows, out_f, in_f, True, True)
    want = layer.product(x, "silu", m, r)
    apart = torch.full((rows, in_f + 5), float("nan"), dtype=torch.bfloat16, device=dev)
    view = apart[:, 3:3 + in_f]
    view.copy_(x)
    assert torch.equal(layer.product(view, "silu", m, r), want)
    x[3, -1] = float("inf")
    y = layer.product(x, "silu", m, r)
    same = torch.arange(rows) != 3
    assert torch.equal(y[same], want[same])


@pytest.mark.parametrize("rows", [1, 9, 33])
@pytest.mark.parametrize("how", ["lanes", "no lanes", "fp32 bias", "packed streams", "decode and multiply"])
def test_products_under_autocast(dev, rows, how):
    """The product is bf16 whatever type autocast would have a library product in: of every way a layer takes, the result without it."""
    layer, w, bias = _layer(dev, 72, 1024, "outlier", bias=True, lanes=how != "no lanes")
    layer._set_shared_buf(torch.empty(layer.N, dtype=torch.bfloat16, device=dev))
    if how == "fp32 bias":
        layer._bias = layer._bias.float()
        layer._bind()
    layer._use_fused = how != "packed streams"
    layer._gemm_ok = how != "decode and multiply"
    x, m, r = _operands(dev, rows, 72, 1024, True, True)
    want = layer.product(x, "silu", m, r)
    _close(want, *ref.epilogue(x, w, bias, "silu", m, r, apart=how != "lanes"))
    for dtype in (torch.float16, torch.bfloat16):
        with torch.autocast("cuda", dtype=dtype):
            got = layer.product(x, "silu", m, r)
            assert torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") is dtype
        assert got.dtype is torch.bfloat16 and torch.equal(got, want)


@pytest.mark.parametrize("lanes", [True, False])
@pytest.mark.parametrize("rows", [1, 33])
def test_products_of_dual_tensors_are_refused(dev, lanes, rows):
    """A tangent is not dropped in silence; other tensors are multiplied inside a forward-mode level as anywhere."""
    from torch.autograd import forward_ad

    layer, _, _ = _layer(dev, 64, 1024, lanes=lanes)
    layer._set_shared_buf(torch.empty(layer.N, dtype=torch.bfloat16, device=dev))
    assert (layer._lanes is not None) == lanes
    given = _operands(dev, rows, 64, 1024, True, True)
    want = layer.product(given[0], "silu", *given[1:])
    with forward_ad.dual_level():
        assert torch.equal(layer.product(given[0], "silu", *given[1:]), want)
        for i in range(3):
            duals = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(given)]
            for grad in (torch.enable_grad, torch.no_grad):
                with grad(), pytest.raises(RuntimeError, match="no gradient"):
                    layer.product(duals[0], "silu", *duals[1:])


def test_prompts_at_a_long_stride_are_taken_in_parts(dev):
    """4096 rows 1 MB apart: a part more than 32-bit offsets hold."""
    layer, w, bias = _layer(dev, 96, 256, "t", bias=True)
    far = torch.zeros((4096, 524672), dtype=torch.bfloat16, device=dev)
    x, m, r = _operands(dev, 4096, 96, 256, True, True)
    far[:, :256] = x
    _close(layer.product(far[:, :256], "silu", m, r), *ref.epilogue(x, w, bias, "silu", m, r))


@pytest.mark.parametrize("out_f,in_f,rows", [(256, 512, 1), (2000, 520, 3), (640, 4608, 7), (1001, 2056, 13), (4096, 11008, 13), (40960, 2048, 3), (4096, 36864, 2),
                                             (72, 1024, 40), (17408, 1024, 100), (12288, 6144, 530), (5126, 5120, 300)])
def test_products_write_over_their_operands(dev, out_f, in_f, rows):
    """The C entry: multiplier and residual may be y itself, and what lies behind the rows stays."""
    import ctypes as C

    from ixrun_amd import _lib

    layer, _, bias = _layer(dev, out_f, in_f, "t" if out_f * in_f > 1 << 22 else "outlier", bias=True)
    x, m, r = _operands(dev, rows, out_f, in_f, True, True)
    need = _lib.lib().ixh_lanes_product_workspace_bytes(layer._lane_ref, rows)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    for pad in (0, 3, 8):
        for over in ("multiplier", "residual", "both"):
            ld = out_f + pad
            held = torch.full((rows + 1, ld), 7.0, dtype=torch.bfloat16, device=dev)
            first, second = (m, r) if over != "both" else (m, m)
            held[:rows, :out_f] = second if over == "residual" else first
            want = layer.product(x, "gelu_tanh", first, second)
            at, other = held.data_ptr(), (r if over == "multiplier" else m)
            ep = _lib.IxhEpilogue(3, at if over != "residual" else other.data_ptr(), ld if over != "residual" else out_f,
                                  at if over != "multiplier" else other.data_ptr(), ld if over != "multiplier" else out_f)
            _lib.check(_lib.lib().ixh_lanes_product(layer._lane_ref, x.data_ptr(), in_f, bias.data_ptr(), rows, C.byref(ep), at, ld, ws.data_ptr(), need,
                                                    _lib.current_stream(dev)))
            assert torch.equal(held[:rows, :out_f], want)
            assert bool((held[rows] == 7).all()) and bool((held[:, out_f:] == 7).all())


@pytest.mark.parametrize("m,out_f,pad", [(1, 1, 0), (3, 300, 5), (70, 1024, 0), (700, 33, 3)])
def test_epilogues_write_over_their_operands(dev, m, out_f, pad):
    import ctypes as C

    from ixrun_amd import _lib

    v, a, b = _operands(dev, m, out_f, out_f, True, True)
    ld = out_f + pad
    want = ref.activation(v.double(), "relu") * a.double() + b.double()
    bound = ref.U16 * want.abs() + 4 * ref.U32 * ((v.double() * a.double()).abs() + b.double().abs())
    for over in range(3):
        held = torch.full((m + 1, ld), 7.0, dtype=torch.bfloat16, device=dev)
        held[:m, :out_f] = (v, a, b)[over]
        at = [held.data_ptr() if over == i else t.data_ptr() for i, t in enumerate((v, a, b))]
        lds = [ld if over == i else out_f for i in range(3)]
        ep = _lib.IxhEpilogue(4, at[1], lds[1], at[2], lds[2])
        _lib.check(_lib.lib().ixh_epilogue(at[0], lds[0], m, out_f, C.byref(ep), held.data_ptr(), ld, _lib.current_stream(dev)))
        _close(held[:m, :out_f].contiguous(), want, bound)
        assert bool((held[m] == 7).all()) and bool((held[:, out_f:] == 7).all())
