"""Routing and the experts' products against their formulas in 64 bits (operator_reference.py has the bounds)."""
import math

import pytest
import torch

import operator_reference as ref
from helpers import calibrated_weight, outlier_weight, student_t_weight

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


# ---- routing ----
def _check_route(logits, top_k, dev, **options):
    from ixrun_amd import route_experts

    bias = options.get("bias")
    on = dict(options, bias=bias.to(dev) if bias is not None else None)
    ids, weights = route_experts(logits.to(dev), top_k, **on)
    want_ids, want = ref.route(logits, top_k, **options)
    assert ids.dtype == torch.int32 and weights.dtype == torch.float32 and ids.shape == want_ids.shape
    assert torch.equal(ids.cpu(), want_ids)
    got = weights.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    # worked out in 64 bits and rounded once to fp32
    assert bool(((got - want).abs() <= 1.001 * ref.U32 * want.abs() + 2.0 ** -149)[~want.isnan()].all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 1, 1), (1, 64, 6), (5, 7, 7), (3, 65, 1), (130, 128, 8), (33, 200, 16), (2, 1024, 64), (9, 500, 3)])
def test_softmax_routing(dev, dtype, tokens, experts, top_k):
    g = torch.Generator().manual_seed(tokens + experts)
    _check_route((torch.randn(tokens, experts, generator=g) * 2).to(dtype), top_k, dev)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize,scale", [(True, 1.0), (False, 2.5)])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("experts,n_groups,top_groups,top_k", [(32, 1, 1, 5), (160, 8, 3, 6), (96, 4, 4, 8), (64, 64, 9, 9), (12, 6, 1, 2)])
def test_routing_options(dev, scoring, renormalize, scale, with_bias, experts, n_groups, top_groups, top_k):
    g = torch.Generator().manual_seed(experts)
    logits = torch.randn(21, experts, generator=g)
    bias = torch.randn(experts, generator=g) * 0.3 if with_bias else None
    _check_route(logits, top_k, dev, scoring=scoring, bias=bias, n_groups=n_groups, top_groups=top_groups, renormalize=renormalize, scale=scale)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("n_groups,top_groups", [(1, 1), (4, 2)])
def test_routing_of_closed_equal_and_odd_logits(dev, scoring, with_bias, n_groups, top_groups):
    """Rows with no open expert, with fewer than are chosen, with equal logits, the largest and smallest values, NaN and infinity."""
    inf, nan, top = math.inf, math.nan, torch.finfo(torch.float32).max
    logits = torch.zeros(12, 16)
    logits[0] = -inf
    logits[1] = -inf
    logits[1, 9] = 0.5
    logits[2, ::2] = 1.0
    logits[3] = -top
    logits[4] = torch.arange(16) % 3 - 1.0
    logits[5, 4] = nan
    logits[6, 3] = inf
    logits[7] = torch.tensor([top, -top] * 8)
    logits[8, 1:] = -0.0
    logits[9, 5:] = -inf
    logits[10] = 300.0 + torch.arange(16)
    logits[11] = -200.0 - torch.arange(16)
    bias = (torch.arange(16) % 5).float() / 8 if with_bias else None
    if with_bias:
        bias[11] = -inf
    _check_route(logits, 4, dev, scoring=scoring, bias=bias, n_groups=n_groups, top_groups=top_groups)


def test_routing_of_views(dev):
    """Leading dimensions, rows at a stride, a transposed view, no tokens at all."""
    from ixrun_amd import route_experts

    g = torch.Generator().manual_seed(3)
    wide = torch.randn(6, 5, 40, generator=g)
    for view in (wide[..., :24], wide[:, 1, 8:30], wide.transpose(0, 1)[..., 1:], wide[2, 2], wide[:, :, :24].transpose(1, 2)):
        on_gpu = wide.to(dev).as_strided(view.shape, view.stride(), view.storage_offset())
        ids, weights = route_experts(on_gpu, 3)
        want_ids, want = ref.route(view, 3)
        assert torch.equal(ids.cpu(), want_ids) and torch.allclose(weights.cpu().double(), want, rtol=1.001 * ref.U32, atol=0)
    ids, weights = route_experts(torch.empty(0, 24, device=dev), 3)
    assert ids.shape == weights.shape == (0, 3)


# ---- the experts' products ----
RECIPES = {"t": student_t_weight, "outlier": outlier_weight, "real": lambda o, i, seed: calibrated_weight(o, i, seed, scale=0.0123046875 / 8)[0]}


def _layer(dev, experts, hidden, inner, recipe="t", level_bits=(3, 5, 8), gated=True, bias=False, activation="silu", seed=0):
    from ixrun_amd import StreamingExperts
    from ixrun_amd.quantize import decode_to_weight, int8x_quantize

    make, rows = RECIPES[recipe], 2 * inner if gated else inner
    gate_up = [int8x_quantize(make(rows, hidden, seed=seed + 2 * e), level_bits) for e in range(experts)]
    down = [int8x_quantize(make(hidden, inner, seed=seed + 2 * e + 1), level_bits) for e in range(experts)]
    g = torch.Generator().manual_seed(seed)
    b1 = (torch.randn(experts, rows, generator=g) * 0.1).bfloat16() if bias else None
    b2 = (torch.randn(experts, hidden, generator=g) * 0.1).bfloat16() if bias else None
    layer = StreamingExperts(gate_up, down, activation=activation, gated=gated, gate_up_bias=b1, down_bias=b2)
    dense = dict(gate_up=torch.stack([decode_to_weight(p) for p in gate_up]).to(dev), down=torch.stack([decode_to_weight(p) for p in down]).to(dev),
                 act=activation, gated=gated, gate_up_bias=b1.to(dev) if bias else None, down_bias=b2.to(dev) if bias else None)
    return layer, dense


def _call(dev, tokens, top_k, experts, hidden, seed=1, skew=0.0, residual=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, hidden, generator=g).bfloat16().to(dev)
    logits = torch.randn(tokens, experts, generator=g) + skew * torch.arange(experts)
    ids = logits.topk(top_k, 1)[1].to(torch.int32).to(dev)
    weights = torch.rand(tokens, top_k, generator=g).to(dev)
    return x, ids, weights, torch.randn(tokens, hidden, generator=g).bfloat16().to(dev) if residual else None


def _close(y, want, bound):
    off = (y.double() - want).abs()
    assert y.dtype == torch.bfloat16 and y.shape == want.shape
    assert bool((off <= bound).all()), f"{int((off > bound).sum())} of {off.numel()} elements, worst {float((off / bound).max()):.2f} bounds"


@pytest.mark.parametrize("recipe,level_bits", [("t", (3, 5, 8)), ("real", (3, 5, 8)), ("outlier", (4, 8)), ("outlier", (3, 4, 5, 6, 8)), ("real", (6, 8))])
@pytest.mark.parametrize("tokens", [1, 2, 7, 40, 150, 700])
def test_experts_by_scheme_and_tokens(dev, recipe, level_bits, tokens):
    layer, dense = _layer(dev, 6, 1024, 320, recipe, level_bits)
    x, ids, weights, residual = _call(dev, tokens, 3, 6, 1024, residual=True)
    _close(layer(x, ids, weights, residual), *ref.experts(x, ids, weights, **dense, residual=residual))


@pytest.mark.parametrize("hidden,inner", [(64, 16), (512, 1), (520, 33), (1, 5), (777, 250), (1400, 744), (96, 1300), (2049, 17), (6000, 40)])
@pytest.mark.parametrize("tokens", [1, 21, 75])
@pytest.mark.parametrize("gated,bias,activation", [(True, True, "gelu_tanh"), (False, False, "relu2")])
def test_experts_by_size(dev, hidden, inner, tokens, gated, bias, activation):
    layer, dense = _layer(dev, 3, hidden, inner, "outlier", gated=gated, bias=bias, activation=activation)
    x, ids, weights, _ = _call(dev, tokens, 2, 3, hidden)
    _close(layer(x, ids, weights), *ref.experts(x, ids, weights, **dense))


@pytest.mark.parametrize("activation", ["none", "silu", "gelu", "gelu_tanh", "relu", "relu2"])
@pytest.mark.parametrize("gated", [True, False])
def test_experts_by_activation(dev, activation, gated):
    layer, dense = _layer(dev, 4, 256, 96, "outlier", gated=gated, activation=activation)
    for tokens in (11, 70):
        x, ids, weights, _ = _call(dev, tokens, 2, 4, 256)
        _close(layer(x, ids, weights), *ref.experts(x, ids, weights, **dense))


@pytest.mark.parametrize("tokens", [100, 250, 390, 512, 513, 700, 1000, 1100])
@pytest.mark.parametrize("level_bits", [(3, 5, 8), (4, 8), (6, 8)])
def test_experts_of_many_tokens(dev, tokens, level_bits):
    """One expert with all of the tokens: tiles of one to 32 blocks of rows, several of them, the last one odd."""
    layer, dense = _layer(dev, 2, 1100, 200, "outlier", level_bits, bias=True)
    x, ids, weights, residual = _call(dev, tokens, 1, 2, 1100, residual=True)
    ids[:] = 1
    ids[-3:] = 0
    _close(layer(x, ids, weights, residual), *ref.experts(x, ids, weights, **dense, residual=residual))


@pytest.mark.parametrize("tokens", [3, 20, 90])
def test_experts_of_uneven_and_missing_places(dev, tokens):
    """All tokens with one expert, experts without any token, places without an expert (whose weights may be anything), tokens of nothing else, an
    expert twice."""
    layer, dense = _layer(dev, 5, 512, 64, "t")
    x, ids, weights, residual = _call(dev, tokens, 3, 5, 512, residual=True)
    ids[:] = 2
    _close(layer(x, ids, weights), *ref.experts(x, ids, weights, **dense))
    x, ids, weights, residual = _call(dev, tokens, 3, 5, 512, skew=2.0, residual=True)
    ids[::2, 1] = -1
    ids[1] = -1
    ids[-1, 0] = 5
    ids[-1, 2] = 2 ** 31 - 1
    clean = torch.where((ids >= 0) & (ids < 5), weights, 0)
    weights = torch.where((ids >= 0) & (ids < 5), weights, math.nan)
    y = layer(x, ids, weights, residual)
    _close(y, *ref.experts(x, ids, clean, **dense, residual=residual))
    assert torch.equal(y[1], residual[1])
    assert torch.equal(layer(x, ids.long(), weights, residual), y)
    far = torch.where(ids < 0, torch.full_like(ids, -1).long() * 2 ** 40, ids.long())
    assert torch.equal(layer(x, far, weights, residual), y)


def test_experts_rows_do_not_hang_on_each_other(dev):
    """A row of infinities and NaN leaves the others as they are, and a token's result is the same wherever it stands."""
    layer, dense = _layer(dev, 4, 512, 64, "real")
    for tokens in (20, 60):
        x, ids, weights, _ = _call(dev, tokens, 2, 4, 512)
        y = layer(x, ids, weights)
        wild = x.clone()
        wild[5] = math.inf
        wild[17, 3] = math.nan
        z = layer(wild, ids, weights)
        same = torch.ones(tokens, dtype=torch.bool)
        same[[5, 17]] = False
        assert torch.equal(z[same], y[same]) and bool(z[17].isnan().all())
        order = torch.randperm(tokens, generator=torch.Generator().manual_seed(2)).to(dev)
        assert torch.equal(layer(x[order], ids[order], weights[order]), y[order])


@pytest.mark.parametrize("tokens", [24, 64])
def test_experts_of_views(dev, tokens):
    layer, _ = _layer(dev, 4, 264, 64, "t")
    x, ids, weights, residual = _call(dev, tokens, 2, 4, 264, residual=True)
    want = layer(x, ids, weights, residual)
    apart = torch.zeros(tokens, 400, dtype=torch.bfloat16, device=dev)
    for start in (0, 1, 3):
        view = apart[:, start:start + 264]
        view.copy_(x)
        assert torch.equal(layer(view, ids, weights, residual), want)
        assert torch.equal(layer(x, ids, weights, view.copy_(residual)), want)
    assert torch.equal(layer(x.t().contiguous().t(), ids.t().contiguous().t(), weights.t().contiguous().t(), residual), want)
    deep = layer(x.view(2, -1, 264), ids.view(2, -1, 2), weights.view(2, -1, 2), residual.view(2, -1, 264))
    assert deep.shape == (2, tokens // 2, 264) and torch.equal(deep.view(tokens, 264), want)
    assert layer(x[:0], ids[:0], weights[:0]).shape == (0, 264)
    # weights of another type are taken as they are
    assert torch.equal(layer(x, ids, weights.bfloat16()), layer(x, ids, weights.bfloat16().float()))


def test_experts_refusals(dev):
    layer, _ = _layer(dev, 2, 64, 16)
    x, ids, weights, residual = _call(dev, 3, 1, 2, 64, residual=True)
    with pytest.raises(TypeError):
        layer(x.float(), ids, weights)
    with pytest.raises(TypeError):
        layer(x, ids.short(), weights)
    with pytest.raises(TypeError):
        layer(x, ids, ids)
    with pytest.raises(ValueError):
        layer(x[:, :63], ids, weights)
    with pytest.raises(ValueError):
        layer(x, ids[:2], weights)
    with pytest.raises(ValueError):
        layer(x, ids, weights[:, :0])
    with pytest.raises(ValueError):
        layer(x, ids, weights, residual[:2])
    with pytest.raises(RuntimeError):
        layer(x.cpu(), ids, weights)
    with pytest.raises(RuntimeError):
        layer(x, ids.cpu(), weights)
    with pytest.raises(RuntimeError, match="no gradient"):
        layer(x.clone().requires_grad_(), ids, weights)
    with pytest.raises(TypeError, match="cast"):
        _layer(dev, 2, 64, 16)[0].float()


def test_experts_state(dev):
    """A state of the same sizes is loaded as a whole; parts of one and lists that do not fit are refused."""
    layer, dense = _layer(dev, 3, 256, 48, "t")
    other, _ = _layer(dev, 3, 256, 48, "t")
    x, ids, weights, _ = _call(dev, 5, 2, 3, 256)
    state = {k: v.clone() for k, v in layer.state_dict().items()}
    for v in other.state_dict().values():
        v.zero_()
    other.load_state_dict(state)
    assert torch.equal(other(x, ids, weights), layer(x, ids, weights))
    other.load_state_dict({k: v.cpu().to(dev) for k, v in state.items()}, assign=True)
    assert torch.equal(other(x, ids, weights), layer(x, ids, weights))
    with pytest.raises(RuntimeError, match="a part of"):
        other.load_state_dict({k: v for k, v in state.items() if k != "_first_pos"}, strict=False)
    wrong = dict(state, _second_off=state["_second_off"] + 1 << 20)
    with pytest.raises(RuntimeError, match="does not fit"):
        other.load_state_dict(wrong)
    assert torch.equal(other(x, ids, weights), layer(x, ids, weights))


@pytest.mark.parametrize("tokens", [1, 33, 200])
def test_experts_from_a_graph_and_another_stream(dev, tokens):
    from ixrun_amd import route_experts

    layer, dense = _layer(dev, 8, 512, 128, "real")
    x, _, _, residual = _call(dev, tokens, 2, 8, 512, residual=True)
    router = torch.randn(8, 512, generator=torch.Generator().manual_seed(4)).to(dev) * 0.05

    def block(x, residual):
        ids, weights = route_experts(x.float() @ router.t(), 2)
        return layer(x, ids, weights, residual=residual), ids, weights

    want = block(x, residual)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = block(x, residual)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, ids, weights = block(x, residual)
    for seed in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)).bfloat16())
        graph.replay()
        eager, eager_ids, _ = block(x, residual)
        torch.cuda.synchronize()
        assert torch.equal(y, eager) and torch.equal(ids, eager_ids)
        _close(y, *ref.experts(x, ids, weights, **dense, residual=residual))


# ---- the same by the kernel that takes a call: slots one by one, tiles of an expert's slots, rows of many cells ----
def _repeated_layer(dev, experts, hidden, inner, recipe, level_bits, distinct=3, **kw):
    """A layer of a few matrices, each with several experts."""
    from ixrun_amd import StreamingExperts
    from ixrun_amd.quantize import decode_to_weight, int8x_quantize

    make, rows = RECIPES[recipe], 2 * inner if kw.get("gated", True) else inner
    gate_up = [int8x_quantize(make(rows, hidden, seed=2 * e), level_bits) for e in range(distinct)]
    down = [int8x_quantize(make(hidden, inner, seed=2 * e + 1), level_bits) for e in range(distinct)]
    of = [e % distinct for e in range(experts)]
    g = torch.Generator().manual_seed(experts)
    b1, b2 = ((torch.randn(experts, n, generator=g) * 0.1).bfloat16() for n in (rows, hidden))
    layer = StreamingExperts([gate_up[e] for e in of], [down[e] for e in of], gate_up_bias=b1, down_bias=b2, **kw)
    stack = lambda packs: torch.stack([decode_to_weight(p).to(dev) for p in packs])[of]
    dense = dict(gate_up=stack(gate_up), down=stack(down), act=kw.get("activation", "silu"), gated=kw.get("gated", True), gate_up_bias=b1.to(dev),
                 down_bias=b2.to(dev))
    return layer, dense


@pytest.mark.parametrize("recipe,level_bits", [("t", (3, 5, 8)), ("real", (3, 5, 8)), ("outlier", (4, 8)), ("real", (6, 8))])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("hidden,inner", [(4100, 40), (8200, 24), (72, 8200), (12301, 9)])
@pytest.mark.parametrize("tokens", [1, 2, 9, 30, 37])
def test_experts_of_long_rows(dev, recipe, level_bits, gated, hidden, inner, tokens):
    layer, dense = _repeated_layer(dev, 12, hidden, inner, recipe, level_bits, gated=gated)
    x, ids, weights, residual = _call(dev, tokens, 3, 12, hidden, skew=0.2, residual=True)
    _close(layer(x, ids, weights, residual), *ref.experts(x, ids, weights, **dense, residual=residual))


@pytest.mark.parametrize("recipe,level_bits", [("t", (3, 5, 8)), ("real", (3, 5, 8)), ("outlier", (4, 8)), ("real", (6, 8))])
@pytest.mark.parametrize("experts,hidden,inner,tokens,top_k", [(24, 2048, 600, 38, 6), (48, 1024, 512, 100, 3), (30, 1001, 515, 62, 5), (24, 2048, 600, 34, 6),
                                                               (30, 1001, 515, 52, 5)])
def test_experts_by_tiles(dev, recipe, level_bits, experts, hidden, inner, tokens, top_k):
    """Up to ten slots an expert, more cells than go one by one; uneven, and with places and tokens of no expert."""
    layer, dense = _repeated_layer(dev, experts, hidden, inner, recipe, level_bits)
    for skew in (0.0, 0.15):
        x, ids, weights, residual = _call(dev, tokens, top_k, experts, hidden, skew=skew, residual=True)
        ids[3, 1:] = -1
        ids[7] = experts
        y = layer(x, ids, weights, residual)
        clean = torch.where((ids >= 0) & (ids < experts), weights, 0)
        _close(y, *ref.experts(x, ids, clean, **dense, residual=residual))
        assert torch.equal(y[7], residual[7])
        wild = x.clone()
        wild[5], wild[17, 3] = math.inf, math.nan
        same = torch.ones(tokens, dtype=torch.bool)
        same[[5, 17]] = False
        assert torch.equal(layer(wild, ids, weights, residual)[same], y[same])


@pytest.mark.parametrize("recipe,level_bits", [("t", (3, 5, 8)), ("real", (3, 5, 8)), ("outlier", (4, 8)), ("real", (6, 8))])
@pytest.mark.parametrize("hidden,inner", [(2048, 1024), (8, 8), (4096, 33), (1037, 520), (4090, 700), (4100, 64), (7160, 130), (8192, 72)])
def test_experts_one_by_one(dev, recipe, level_bits, hidden, inner):
    """Slots by themselves: rows of one to eight cells, the same expert in several slots and twice in a token, places without one, rows of any
    alignment, a row of infinities beside others."""
    layer, dense = _repeated_layer(dev, 9, hidden, inner, recipe, level_bits)
    for tokens, top_k in ((1, 1), (1, 9), (3, 4), (8, 2)):
        x, ids, weights, residual = _call(dev, tokens, top_k, 9, hidden, seed=tokens + top_k, residual=True)
        if tokens > 1:
            ids[0] = 4
            ids[1, 0] = -7
        clean = torch.where(ids >= 0, weights, 0)
        y = layer(x, ids, weights, residual)
        _close(y, *ref.experts(x, ids, clean, **dense, residual=residual))
        apart = torch.zeros(tokens, hidden + 9, dtype=torch.bfloat16, device=dev)
        for start in (1, 8):
            view = apart[:, start:start + hidden]
            view.copy_(x)
            assert torch.equal(layer(view, ids, weights, residual), y)
        if tokens > 1:
            wild = x.clone()
            wild[1] = math.inf
            same = torch.arange(tokens) != 1
            assert torch.equal(layer(wild, ids, weights, residual)[same], y[same])


def test_routing_refusals(dev):
    from ixrun_amd import route_experts

    logits = torch.zeros(3, 16, device=dev)
    for wrong in (dict(top_k=17), dict(top_k=2 ** 32 + 2), dict(top_k=2, n_groups=2 ** 32 + 1, top_groups=1), dict(top_k=2, n_groups=4, top_groups=2 ** 32 + 1),
                  dict(top_k=-1), dict(top_k=2, scoring="max"), dict(top_k=2, bias=torch.zeros(15, device=dev))):
        with pytest.raises((ValueError, RuntimeError)):
            route_experts(logits, **wrong)
    with pytest.raises(TypeError):
        route_experts(logits.double(), 2)
    with pytest.raises(RuntimeError, match="no gradient"):
        route_experts(logits.clone().requires_grad_(), 2)


def test_experts_off_the_gpu_are_refused(dev):
    layer, _ = _layer(dev, 3, 64, 16)
    x, ids, weights, _ = _call(dev, 3, 1, 3, 64)
    want = layer(x, ids, weights)
    layer.cpu()
    for on in ("cpu", dev):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            layer(x.to(on), ids.to(on), weights.to(on))
    layer.to(dev)
    assert torch.equal(layer(x, ids, weights), want)


def test_experts_after_a_refused_cast_and_copied(dev):
    """A refused cast leaves the layer as it was; a copy has weights of its own."""
    import copy

    layer, _ = _layer(dev, 3, 64, 16, bias=True)
    x, ids, weights, _ = _call(dev, 5, 2, 3, 64)
    want = layer(x, ids, weights)
    for cast in (lambda: layer.float(), lambda: layer.half(), lambda: layer.to(torch.float64)):
        with pytest.raises(TypeError, match="cast"):
            cast()
    torch.randn(1 << 20, device=dev)  # (what might take freed memory)
    assert torch.equal(layer(x, ids, weights), want)
    other = copy.deepcopy(layer)
    for t in layer.state_dict().values():
        t.zero_()
    assert torch.equal(other(x, ids, weights), want)


def test_experts_states_of_other_types_are_refused(dev):
    layer, _ = _layer(dev, 3, 256, 48, "t", bias=True)
    x, ids, weights, _ = _call(dev, 5, 2, 3, 256)
    want = layer(x, ids, weights)
    state = {k: v.clone() for k, v in layer.state_dict().items()}
    changes = dict(_first_plane=lambda t: t.to(torch.int8), _first_pos=lambda t: t.int(), _second_off=lambda t: t.long(), _second_scale=lambda t: t.float(),
                   _first_val=lambda t: t[:-64], _first_bias=lambda t: t.t().contiguous().t(), _second_bias=lambda t: t.float())
    for name, change in changes.items():
        with pytest.raises(RuntimeError, match=name):
            layer.load_state_dict(dict(state, **{name: change(state[name])}), assign=True)
        assert torch.equal(layer(x, ids, weights), want)


def test_experts_of_a_long_call_are_taken_in_parts(dev, monkeypatch):
    from ixrun_amd import experts

    layer, dense = _layer(dev, 4, 264, 64, "t")
    x, ids, weights, residual = _call(dev, 71, 2, 4, 264, residual=True)
    for most in (1, 7, 60, 100):
        monkeypatch.setattr(experts, "MOST_PLACES", most)
        _close(layer(x, ids, weights, residual), *ref.experts(x, ids, weights, **dense, residual=residual))


def test_experts_write_over_their_input(dev):
    """The C entry: y may be the residual or x, and what lies behind the rows stays."""
    import ctypes as C

    from ixrun_amd import _lib

    layer, _ = _layer(dev, 4, 264, 64, "t")
    for tokens in (1, 9, 60):
        x, ids, weights, residual = _call(dev, tokens, 2, 4, 264, residual=True)
        want = layer(x, ids, weights, residual)
        need = _lib.lib().ixh_experts_workspace_bytes(C.byref(layer._struct), tokens, 2)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        for over_x in (False, True):
            held = torch.full((tokens + 1, 280), 7.0, dtype=torch.bfloat16, device=dev)
            held[:tokens, :264] = x if over_x else residual
            a, r = (held, residual) if over_x else (x, held)
            _lib.check(_lib.lib().ixh_experts(C.byref(layer._struct), a.data_ptr(), a.stride(0), tokens, ids.data_ptr(), weights.data_ptr(), 2, r.data_ptr(),
                                              r.stride(0), held.data_ptr(), 280, ws.data_ptr(), need, _lib.current_stream(dev)))
            assert torch.equal(held[:tokens, :264], want)
            assert bool((held[tokens] == 7).all()) and bool((held[:, 264:] == 7).all())


def test_two_calls_at_once_and_graphs_in_turn(dev):
    """Calls of two streams side by side, and two graphs of one layer replayed in turn, with other work in between."""
    layer, dense = _layer(dev, 8, 512, 128, "real")
    calls = [_call(dev, tokens, 3, 8, 512, seed=tokens, residual=True) for tokens in (1, 40, 300)]
    want = [layer(*c) for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        got = []
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(layer(*c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(layer(*c))
    for turn in range(4):
        for y in outs:
            y.zero_()
        for g in (graphs if turn % 2 else graphs[::-1]):
            g.replay()
            layer(*calls[turn % 3])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_dual_tensors_are_refused(dev):
    """A tangent is not dropped in silence; other tensors are routed and multiplied inside a forward-mode level as anywhere."""
    from torch.autograd import forward_ad

    from ixrun_amd import route_experts

    layer, _ = _layer(dev, 4, 64, 16)
    x, ids, weights, residual = _call(dev, 3, 2, 4, 64, residual=True)
    logits, bias = torch.randn(3, 4, device=dev), torch.randn(4, device=dev)
    want, routed = layer(x, ids, weights, residual), route_experts(logits, 2, bias=bias)
    with forward_ad.dual_level():
        assert torch.equal(layer(x, ids, weights, residual), want)
        assert all(torch.equal(a, b) for a, b in zip(route_experts(logits, 2, bias=bias), routed))
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        calls = [lambda: layer(dual(x), ids, weights, residual), lambda: layer(x, ids, dual(weights), residual), lambda: layer(x, ids, weights, dual(residual)),
                 lambda: route_experts(dual(logits), 2), lambda: route_experts(logits, 2, bias=dual(bias))]
        for call in calls:
            for grad in (torch.enable_grad, torch.no_grad):
                with grad(), pytest.raises(RuntimeError, match="no gradient"):
                    call()


def _experts_of_columns(x, ids, weights, residual, gate_up, down, gate_up_bias, down_bias):
    """ref.experts of gated ReLU experts, over those columns of x and of the intermediate that are not 0 everywhere."""
    y = torch.zeros(x.shape[0], down.shape[1], dtype=torch.float64, device=x.device)
    off, size = torch.zeros_like(y), torch.zeros_like(y)
    for e in range(down.shape[0]):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        (g, dg), (u, du) = (ref.product(x[t], w, b) for w, b in zip(gate_up[e].chunk(2), gate_up_bias[e].chunk(2)))
        a, da = ref.activated(g, dg, "relu")
        h, dh = ref.rounded(a * u, da * (u.abs() + du) + a.abs() * du + ref.U32 * (a * u).abs())
        v, dv = ref.product(h, down[e], down_bias[e])
        dv = dv + dh @ down[e].double().abs().t()
        w = weights[t, j].double().unsqueeze(1)
        y.index_add_(0, t, w * v)
        off.index_add_(0, t, w.abs() * dv)
        size.index_add_(0, t, (w * v).abs())
    y = y + residual.double()
    off = off + (ids.shape[1] + 2) * ref.U32 * size + ref.U32 * y.abs()
    return y, off + ref.U16 * (y.abs() + off)


@pytest.mark.parametrize("recipe,level_bits", [("t", (3, 5, 8)), ("outlier", (4, 8)), ("real", (3, 5, 8)), ("real", (6, 8))])
@pytest.mark.parametrize("hidden,inner", [(32767, 16), (32768, 8), (33001, 24), (66000, 9), (24, 33001), (16, 66048)])
def test_experts_of_rows_whose_positions_start_over(dev, recipe, level_bits, hidden, inner):
    """Rows of 64 cells and more, where a list's positions count from column 32768 n on and places without an element point at 0: slots by
    themselves, tiles of a few, and many tokens to an expert.  All columns but a hundred of the long rows are 0, which adds nothing to a sum and
    so nothing to its bound: an element that is multiplied with another column's activation is far outside."""
    layer, dense = _repeated_layer(dev, 4, hidden, inner, recipe, level_bits, distinct=2, activation="relu")
    long = max(hidden, inner)
    borders = [c + d for c in (0, 512, 32256, 32768, 33280, 65536, long) for d in (-2, -1, 0, 1, 31)]
    some = torch.randperm(long, generator=torch.Generator().manual_seed(long))[:70].tolist()
    at = torch.tensor(sorted({c for c in borders + some if 0 <= c < long}), device=dev)
    none = torch.ones(long, dtype=torch.bool, device=dev)
    none[at] = False
    gate_up, down, bias = dense["gate_up"], dense["down"], layer._first_bias
    if hidden == long:
        gate_up = gate_up[:, :, at]
    else:  # the gate is closed elsewhere
        bias[:, :inner][:, none] = -1000.0
        both = torch.cat([at, at + inner])
        gate_up, down, bias = gate_up[:, both], down[:, :, at], bias[:, both]
    for tokens, top_k in ((1, 2), (9, 3), (21, 2), (30, 2)):
        x, ids, weights, residual = _call(dev, tokens, top_k, 4, hidden, seed=tokens, residual=True)
        if hidden == long:
            x[:, none] = 0.0
        y = layer(x, ids, weights, residual)
        _close(y, *_experts_of_columns(x[:, at] if hidden == long else x, ids, weights, residual, gate_up, down, bias, dense["down_bias"]))
        if tokens > 1:  # the column that places without an element point at, too
            x[tokens // 2, 0] = math.inf
            same = torch.arange(tokens) != tokens // 2
            assert torch.equal(layer(x, ids, weights, residual)[same], y[same])


@pytest.mark.parametrize("recipe,level_bits", [("t", (3, 5, 8)), ("real", (3, 5, 8)), ("outlier", (4, 8)), ("real", (6, 8))])
@pytest.mark.parametrize("hidden,inner,top_k", [(264, 100, 16), (100, 40, 13), (72, 8000, 1), (520, 2000, 4), (1037, 700, 7), (40, 3000, 2)])
def test_experts_whose_sum_is_in_the_second_launch(dev, recipe, level_bits, hidden, inner, top_k):
    """Up to sixteen cells of a token's slots in one workgroup, and calls of more tokens than that is done for: the same sums."""
    layer, dense = _repeated_layer(dev, 16, hidden, inner, recipe, level_bits)
    for tokens in (1, 2, 5, 40):
        x, ids, weights, residual = _call(dev, tokens, top_k, 16, hidden, seed=tokens, residual=True)
        if tokens > 1:
            ids[0] = 4
            ids[1, 0] = -7
        clean = torch.where(ids >= 0, weights, 0)
        y = layer(x, ids, torch.where(ids >= 0, weights, math.nan), residual)
        _close(y, *ref.experts(x, ids, clean, **dense, residual=residual))
        _close(layer(x, ids, weights), *ref.experts(x, ids, clean, **dense))
        for t in range(min(tokens, 3)):
            _close(layer(x[t:t + 1], ids[t:t + 1], weights[t:t + 1], residual[t:t + 1]), *ref.experts(x[t:t + 1], ids[t:t + 1], clean[t:t + 1], **dense,
                                                                                                 residual=residual[t:t + 1]))
