"""Routing of tokens to experts, and the experts' products over packed weights.

A layer of experts has a feed-forward block for each expert, of which a token takes the few that its router chooses.
``route_experts`` makes that choice from the router's logits; ``StreamingExperts`` keeps all experts' weights packed on the
GPU, in the lane layout that ``StreamingLinear`` multiplies from (``csrc/ixh_lanes.h``), and reads those of the experts that
some token has chosen.  Both serve inference, as the packed layers do.  The reference has no counterpart.
"""
from __future__ import annotations

import ctypes as C

import torch
import torch.nn as nn

from . import _lib
from .config import DEFAULT_LEVELS, FUSED_TILE
from .quantize import quantize_for_deploy

__all__ = ["StreamingExperts", "route_experts"]

LOGIT_TYPES = {torch.float32: _lib.IXH_F32, torch.float16: _lib.IXH_F16, torch.bfloat16: _lib.IXH_BF16}
SCORINGS = {"softmax": _lib.IXH_SCORE_SOFTMAX, "sigmoid": _lib.IXH_SCORE_SIGMOID}
MOST_EXPERTS = 1024
MOST_PLACES = 1 << 17  # tokens times experts of each in one call of the library: bounds the call's scratch (4 bytes a column of each: 3.8 GB at 7168)


def route_experts(logits, top_k: int, *, scoring: str = "softmax", bias=None, n_groups: int = 1, top_groups: int | None = None,
                  renormalize: bool = True, scale: float = 1.0):
    """The experts of each token and their weights: ``(ids int32 [..., top_k], weights fp32 [..., top_k])``, best first.

    ``logits`` [..., experts] in fp32, fp16 or bf16.  The scores are their ``softmax`` or ``sigmoid``.  Without a ``bias`` the largest
    logits are chosen, with one (fp32 [experts], as a load-balanced router has) the largest ``score + bias``, formed in 64 bits; equal ones
    go to the lowest index.  With ``n_groups`` the experts are that many runs of equal length, and the choice is among the ``top_groups``
    best: those with the largest choice, or, with a bias, the largest sum of two.  The weights are the scores of the chosen experts,
    divided by their sum with ``renormalize``, times ``scale``.

    A logit of -infinity closes its expert for the token (all of them for a token of padding); a place that finds no open expert has id -1
    and weight 0, which ``StreamingExperts`` passes over.  A NaN is chosen first and reaches the weights."""
    top_groups = n_groups if top_groups is None else top_groups
    done = _lib.host().route(logits, bias, top_k, n_groups, top_groups, SCORINGS.get(scoring), renormalize, scale)
    if done is not None:
        return done
    _lib.inference_only("route_experts", logits, bias)
    if not logits.is_cuda:
        raise RuntimeError(f"logits must live on the GPU (got {logits.device}); the HIP path has no CPU fallback")
    if logits.dtype not in LOGIT_TYPES:
        raise TypeError(f"logits must be fp32, fp16 or bf16 (got {logits.dtype})")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits need a last dimension of experts")
    if scoring not in SCORINGS:
        raise ValueError(f"scoring {scoring!r} is none of {sorted(SCORINGS)}")
    experts, dev = logits.shape[-1], logits.device
    rows = logits.reshape(-1, experts) if logits.dim() != 2 else logits
    if rows.stride(1) != 1 or (rows.shape[0] > 1 and rows.stride(0) < experts):
        rows = rows.contiguous()
    if bias is not None:
        if bias.device != dev or bias.numel() != experts:
            raise ValueError(f"bias must hold {experts} elements on {dev}")
        bias = bias.to(torch.float32).contiguous()
    if not (0 <= top_k <= experts and 0 <= n_groups <= experts and 0 <= top_groups <= experts):  # (as 32-bit numbers they might pass)
        raise ValueError(f"top_k {top_k}, n_groups {n_groups} or top_groups {top_groups} of {experts} experts")
    routing = _lib.IxhRouting(experts, top_k, n_groups, top_groups, SCORINGS[scoring], bool(renormalize), scale)
    shape = logits.shape[:-1] + (max(top_k, 0),)
    ids = torch.empty(shape, dtype=torch.int32, device=dev)
    weights = torch.empty(shape, dtype=torch.float32, device=dev)
    with _lib.on_device(dev):
        _lib.check(_lib.lib().ixh_route(C.byref(routing), rows.data_ptr(), LOGIT_TYPES[logits.dtype], rows.stride(0), rows.shape[0],
                                        bias.data_ptr() if bias is not None else None, ids.data_ptr(), weights.data_ptr(),
                                        _lib.current_stream(dev)))
    return ids, weights


LAYOUT = ("plane", "off", "pos", "val", "scale")


class StreamingExperts(nn.Module):
    """A layer of experts over packed weights: ``y = residual + sum_j weights[:, j] * down_e(act(gate_e x) * up_e x)``, ``e = ids[:, j]``.

    ``gate_up`` and ``down`` are lists of packed dictionaries (``int8x_quantize``), one for each expert: ``[2 * inner, hidden]`` with the
    gate's rows first (``[inner, hidden]`` if not ``gated``) and ``[hidden, inner]``; ``from_weights`` packs bf16 tensors.  Biases are
    ``[n_experts, 2 * inner]`` and ``[n_experts, hidden]``.  All experts' weights stay on the GPU in the lane layout, which holds the same
    integers; the packed streams are not kept.  Weights are ``bf16(value * scale)`` as in every other product, the intermediate is rounded
    to bf16, sums are fp32.
    """

    def __init__(self, gate_up: list, down: list, *, activation: str | None = "silu", gated: bool = True, gate_up_bias=None, down_bias=None):
        super().__init__()
        if not gate_up or len(gate_up) != len(down):
            raise ValueError(f"{len(gate_up)} and {len(down)} matrices: one of each for every expert")
        if len(gate_up) > MOST_EXPERTS:
            raise ValueError(f"{len(gate_up)} experts, {MOST_EXPERTS} at most")
        if activation not in _lib.ACTIVATIONS:
            raise ValueError(f"activation {activation!r} is none of {[a for a in _lib.ACTIVATIONS if a]}")
        self.n_experts, self.gated, self.activation = len(gate_up), bool(gated), activation
        self.hidden, self.inner = down[0]["out_f"], down[0]["in_f"]
        rows = 2 * self.inner if gated else self.inner
        for name, packed, shape in (("gate_up", gate_up, (rows, self.hidden)), ("down", down, (self.hidden, self.inner))):
            if any((p["out_f"], p["in_f"]) != shape or tuple(p["level_bits"]) != tuple(packed[0]["level_bits"]) for p in packed):
                raise ValueError(f"{name} must be {shape[0]} x {shape[1]} of the same levels for every expert")
        dev = torch.device("cuda", torch.cuda.current_device())
        self._lay_out("first", gate_up, dev, interleave=gated)
        self._lay_out("second", down, dev)
        for name, b, width in (("first", gate_up_bias, rows), ("second", down_bias, self.hidden)):
            if b is not None:
                if tuple(b.shape) != (self.n_experts, width):
                    raise ValueError(f"a bias of {tuple(b.shape)}, expected {(self.n_experts, width)}")
                b = b.detach().to(device=dev, dtype=torch.bfloat16).clone().contiguous()
            self.register_buffer(f"_{name}_bias", b)
        self._bind()

    @classmethod
    def from_weights(cls, gate_up, down, level_bits=DEFAULT_LEVELS, **kw) -> "StreamingExperts":
        """From bf16 weights ``[n_experts, 2 * inner, hidden]`` and ``[n_experts, hidden, inner]``, each expert's matrices packed for themselves."""
        pack = lambda ws: [quantize_for_deploy(w, level_bits) for w in ws]
        return cls(pack(gate_up), pack(down), **kw)

    @torch.no_grad()
    def _lay_out(self, name: str, packed: list, dev, interleave: bool = False) -> None:
        """One matrix of all experts in the lane layout: ``plane`` [experts, words], ``off`` [experts, cells + 1], one list."""
        L, stream = _lib.lib(), _lib.current_stream(dev)
        n_rows, in_f = packed[0]["out_f"], packed[0]["in_f"]
        half = -(-n_rows // 2 // 16) * 16 if interleave else 0
        out_f = 2 * half if interleave else n_rows
        bits = _lib.lane_bits(packed[0]["level_bits"], [sum(c) for c in zip(*(p["counts"] for p in packed))])
        words, cells, n = L.ixh_lanes_plane_words(out_f, in_f, bits), L.ixh_lanes_cells(out_f, in_f), len(packed)
        if words < 0:
            raise ValueError(f"{n_rows} x {in_f} has no lane layout")
        scale = torch.stack([p["scale"].reshape(()).to(dev) for p in packed])
        if not bool((scale.float().abs() * 127 < 2.0 ** 128 - 2.0 ** 119).all()):
            raise ValueError("a scale of which some weights are infinite: the lane layout holds none")
        plane = torch.empty((n, words), dtype=torch.int32, device=dev)
        off = torch.zeros((n, cells + 1), dtype=torch.int32, device=dev)
        quads = torch.empty((n, cells), dtype=torch.int32, device=dev)

        def weights(p):
            dp = p.get("device_packed")
            if dp is None or dp.device != dev:
                dp = _lib.DevicePacked.from_dict(p, dev)
            table = p.get("table512")
            w = torch.empty(dp.N, dtype=torch.bfloat16, device=dev)
            dp.decode(table.to(dev) if table is not None else dp.prefix_build(FUSED_TILE), FUSED_TILE, out_bf16=w)
            if not interleave:
                return w
            both = torch.zeros((2, half, in_f), dtype=torch.bfloat16, device=dev)
            both[:, : n_rows // 2] = w.view(2, n_rows // 2, in_f)
            return both.view(2, half // 16, 16, in_f).transpose(0, 1).contiguous()

        def layout(e, *lists):
            return _lib.IxhLanes(bits, out_f, in_f, plane[e].data_ptr(), words, *lists, scale[e].data_ptr())

        for e, p in enumerate(packed):
            w = weights(p)
            _lib.check(L.ixh_lanes_pack(w.data_ptr(), C.byref(layout(e, None, None, None, 0)), quads[e].data_ptr(), stream))
        torch.cumsum(quads, 1, dtype=torch.int32, out=off[:, 1:])
        held = [max(-(-t // 64) * 64, 64) for t in off[:, -1].tolist()]  # whole groups, the one synchronisation
        if sum(held) >= 1 << 30:
            raise ValueError("more listed elements than a layout holds")
        pos = torch.empty(4 * sum(held), dtype=torch.int16, device=dev)
        val = torch.zeros(4 * sum(held), dtype=torch.int8, device=dev)
        at = 0
        for e, p in enumerate(packed):
            w = weights(p)
            part = layout(e, off[e].data_ptr(), pos[4 * at:].data_ptr(), val[4 * at:].data_ptr(), held[e])
            _lib.check(L.ixh_lanes_list(w.data_ptr(), C.byref(part), stream))
            off[e] += at
            at += held[e]
        for part, t in zip(LAYOUT, (plane, off, pos, val, scale)):
            self.register_buffer(f"_{name}_{part}", t)

    def _matrix(self, name: str, out_f: int, in_f: int):
        plane, off, pos, val, scale = (getattr(self, f"_{name}_{part}") for part in LAYOUT)
        bias = getattr(self, f"_{name}_bias")
        for t in (plane, off, pos, val, scale) + ((bias,) if bias is not None else ()):
            _lib._require_cuda(t, "an experts' layout")
        bits = plane.shape[1] // (_lib.lib().ixh_lanes_plane_words(out_f, in_f, 8) // 8)
        return _lib.IxhExpertMatrix(bits, out_f, in_f, plane.data_ptr(), plane.numel(), off.data_ptr(), pos.data_ptr(), val.data_ptr(),
                                    pos.numel() // 4, scale.data_ptr(), bias.data_ptr() if bias is not None else None)

    def _bind(self):
        """Point the library's arguments at the buffers; those of a layer that is not on a GPU are none."""
        self._struct, self._struct_at = None, 0
        if not self._first_plane.is_cuda:
            return
        rows = -(-self.inner // 16) * 32 if self.gated else self.inner
        self._struct = _lib.IxhExperts(self.n_experts, self.gated, _lib.ACTIVATIONS[self.activation], self.hidden, self.inner,
                                       self._matrix("first", rows, self.hidden), self._matrix("second", self.hidden, self.inner))
        self._struct_at, self._device_index = C.addressof(self._struct), self._first_plane.device.index

    def __getstate__(self):
        return {**self.__dict__, "_struct": None, "_struct_at": 0}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._bind()

    def _apply(self, fn, recurse=True):
        # .to() may move the buffers: point the arguments at the new storage.  (Their types are the layout's and stay.)
        kept = dict(self.named_buffers(recurse=False))
        out = super()._apply(fn, recurse)
        cast = [name for name, t in kept.items() if getattr(self, name).dtype != t.dtype]
        if cast:
            for name, t in kept.items():
                setattr(self, name, t)
            raise TypeError(f"an experts' layer cannot be cast: {cast[0]} is {kept[cast[0]].dtype}")
        self._bind()
        return out

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        """A layout is loaded as a whole, and only one whose lists the kernels can read within their buffers."""
        for name in ("first", "second"):
            keys = [f"{prefix}_{name}_{part}" for part in LAYOUT]
            given = [k for k in keys if k in state_dict]
            if given and len(given) != len(keys):
                error_msgs.append(f"a part of an experts' layout: {[k for k in keys if k not in state_dict]} are missing")
                return
            for k, part in zip(given, LAYOUT):
                t, own = state_dict[k], getattr(self, f"_{name}_{part}")
                if t.dtype != own.dtype or t.shape != own.shape or not t.is_contiguous():
                    error_msgs.append(f"{k} is {t.dtype} {tuple(t.shape)}, expected {own.dtype} {tuple(own.shape)}, contiguous")
                    return
            if given:
                off, pos = state_dict[keys[1]], state_dict[keys[2]]
                if bool((off[:, 1:] < off[:, :-1]).any()) or int(off[:, 0].min()) < 0 or int(off[:, -1].max()) > pos.numel() // 4:
                    error_msgs.append(f"{keys[1]} does not fit the list")
                    return
            k, own = f"{prefix}_{name}_bias", getattr(self, f"_{name}_bias")
            if own is not None and k in state_dict and (state_dict[k].dtype != own.dtype or state_dict[k].shape != own.shape or not state_dict[k].is_contiguous()):
                error_msgs.append(f"{k} is {state_dict[k].dtype} {tuple(state_dict[k].shape)}, expected {own.dtype} {tuple(own.shape)}, contiguous")
                return
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        self._bind()

    def extra_repr(self) -> str:
        return f"experts={self.n_experts}, hidden={self.hidden}, inner={self.inner}, gated={self.gated}, activation={self.activation}"

    def _rows(self, t, what: str, shape):
        if t.dtype is not torch.bfloat16:
            raise TypeError(f"{what} must be bf16 (got {t.dtype})")
        if t.device != self._first_plane.device:
            raise RuntimeError(f"{what} must live on {self._first_plane.device} (got {t.device}); the HIP path has no CPU fallback")
        if t.shape != shape:
            raise ValueError(f"{what} is {tuple(t.shape)}, expected {tuple(shape)}")
        rows = t.reshape(-1, self.hidden) if t.dim() != 2 else t
        return rows if rows.stride(1) == 1 and (rows.shape[0] <= 1 or rows.stride(0) >= self.hidden) else rows.contiguous()

    def forward(self, x, ids, weights, residual=None):
        """``x`` bf16 [..., hidden]; ``ids`` (int32 or int64) and ``weights`` [..., top_k] as ``route_experts`` gives them; ``residual`` like ``x``.

        A place whose id is no expert's adds nothing."""
        if self._struct_at:
            y = _lib.host().experts(self._struct_at, self._device_index, MOST_PLACES, x, ids, weights, residual)
            if y is not None:
                return y
        _lib.inference_only("StreamingExperts", x, weights, residual)
        if self._struct is None:
            raise RuntimeError(f"the layer is on {self._first_plane.device}; the HIP path has no CPU fallback")
        dev = self._first_plane.device
        if x.dim() < 1 or x.shape[-1] != self.hidden:
            raise ValueError(f"x is {tuple(x.shape)}, expected [..., {self.hidden}]")
        rows = self._rows(x, "x", x.shape)
        if ids.dim() != x.dim() or ids.shape[:-1] != x.shape[:-1] or ids.shape != weights.shape or ids.shape[-1] < 1:
            raise ValueError(f"ids {tuple(ids.shape)} and weights {tuple(weights.shape)} must be {tuple(x.shape[:-1])} by the experts of a token")
        if ids.dtype not in (torch.int32, torch.int64) or not weights.is_floating_point():
            raise TypeError(f"ids must be int32 or int64 and weights floating-point (got {ids.dtype}, {weights.dtype})")
        if ids.device != dev or weights.device != dev:
            raise RuntimeError(f"ids and weights must live on {dev} (got {ids.device}, {weights.device})")
        if ids.dtype is torch.int64:
            ids = ids.clamp(-1, self.n_experts).to(torch.int32)
        ids, weights = ids.contiguous(), weights.to(torch.float32).contiguous()
        res = self._rows(residual, "residual", x.shape) if residual is not None else None
        n, top_k = rows.shape[0], ids.shape[-1]
        y = torch.empty(x.shape, dtype=torch.bfloat16, device=dev)
        step = max(MOST_PLACES // top_k, 1)
        L = _lib.lib()
        with _lib.on_device(dev):
            need = L.ixh_experts_workspace_bytes(C.byref(self._struct), min(n, step), top_k)
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            for t in range(0, n, step):
                _lib.check(L.ixh_experts(C.byref(self._struct), rows.data_ptr() + 2 * t * rows.stride(0), rows.stride(0), min(step, n - t),
                                         ids.data_ptr() + 4 * t * top_k, weights.data_ptr() + 4 * t * top_k, top_k,
                                         res.data_ptr() + 2 * t * res.stride(0) if res is not None else None,
                                         res.stride(0) if res is not None else 0, y.data_ptr() + 2 * t * self.hidden, self.hidden,
                                         ws.data_ptr(), need, _lib.current_stream(dev)))
        return y
