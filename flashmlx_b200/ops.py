"""Python mirror of the reference's operator calls, running on libflashmoe.

Same names, argument meaning and error behaviour as the MLX calls the reference makes
(server/src/model.cpp):

    quantized_matmul(x, w, scales, biases, transpose=True, group_size=64, bits=4)
        <- mx::quantized_matmul                                   model.cpp:476-480
    gather_qmm(x, w, scales, biases, lhs_indices, rhs_indices, transpose=True,
               group_size=64, bits=4, sorted_indices=False)
        <- mx::gather_qmm                                         model.cpp:703-721
    MoEBlock(config, weights)(x)
        <- LlamaModel::moe_block                                  model.cpp:750-807

Tensors are torch CUDA tensors used only as device buffers: bf16 activations,
uint32 (or int32) packed weights, bf16 scales / biases.  Work is queued on torch's
current stream.  Unsupported arguments raise ValueError / NotImplementedError before
any launch, like MLX's argument checks; device-side failures raise FlashMoEError at
the next `synchronize()`.
"""
from __future__ import annotations

import ctypes as C
import functools
import threading
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import FlashMoEError, MoEConfig, MoEOutputs, MoEWeights, QWeight

__all__ = ["Handle", "default_handle", "quantized_matmul", "gather_qmm", "MoEConfig", "MoEWeightsT", "MoEBlock",
           "FlashMoEError", "synchronize", "bf16_from_numpy", "u32_from_numpy", "bf16_to_numpy"]

_tls = threading.local()


def _raw_stream(device: int) -> int:
    """The current stream's cudaStream_t, without a torch.cuda.Stream object where torch offers it."""
    return torch.cuda.current_stream(device).cuda_stream


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


class Handle:
    """One libflashmoe handle (device workspace + stream binding)."""

    _stream = None  # the stream fm_set_stream was last given (None: not by bind_stream)

    def __init__(self, device: int | None = None):
        self.lib = _lib.load()
        if device is None:
            device = torch.cuda.current_device()
        self.device = device
        h = C.c_void_p()
        with torch.cuda.device(device):
            st = self.lib.fm_create(C.byref(h), device, C.c_void_p(torch.cuda.current_stream().cuda_stream))
        if st != _lib.FM_OK:
            raise FlashMoEError(st, "fm_create failed: " + self.lib.fm_status_string(st).decode())
        self.h = h

    def close(self):
        if self.h and not getattr(self, "_borrowed", False):  # a borrowed view never destroys
            self.lib.fm_destroy(self.h)
        self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def check(self, st: int):
        if st != _lib.FM_OK:
            raise FlashMoEError(st, self.lib.fm_last_error(self.h).decode())

    def bind_stream(self, stream: torch.cuda.Stream | None = None):
        s = stream if stream is not None else torch.cuda.current_stream(self.device)
        self.check(self.lib.fm_set_stream(self.h, C.c_void_p(s.cuda_stream)))
        self._stream = s.cuda_stream

    def bind_current(self):
        """bind_stream() to torch's current stream, told to the library only when it changes (for
        handles that nothing else binds: a call's host time is a few microseconds)."""
        s = _raw_stream(self.device)
        if s != self._stream or getattr(self, "_borrowed", False):
            self.check(self.lib.fm_set_stream(self.h, s))
            self._stream = s

    def set_path(self, path: int):
        self.check(self.lib.fm_set_path(self.h, path))

    def last_path(self) -> int:
        """FM_PATH_GEMV (1) or FM_PATH_TCGEN05 (2): the expert-product path of the
        handle's last call, i.e. which of MLX's two arithmetic forms it followed."""
        return int(self.lib.fm_last_path(self.h))

    def set_route_mode(self, mode: int):
        """FM_ROUTE_GRID (cooperative, grid barriers) or FM_ROUTE_LAST_BLOCK (batches of
        at most 128 tokens: top-k, sort and planning in the block that finishes the router
        GEMV last); FM_ROUTE_AUTO is the grid form."""
        self.check(self.lib.fm_set_route_mode(self.h, mode))

    def sync(self):
        self.check(self.lib.fm_sync_status(self.h))

    def workspace_bytes(self) -> int:
        return int(self.lib.fm_workspace_bytes(self.h))

    def profile(self, on: bool = True):
        self.check(self.lib.fm_profile_enable(self.h, int(on)))

    def profile_report(self, reset: bool = True) -> dict:
        """{kernel name: (launches, total device ms)} since the last reset."""
        buf = (_lib.KernelTime * 32)()
        n = C.c_int(0)
        self.check(self.lib.fm_profile_report(self.h, buf, 32, C.byref(n), int(reset)))
        return {buf[i].name.decode(): (int(buf[i].launches), float(buf[i].total_ms)) for i in range(min(n.value, 32))}


def default_handle(device: int | None = None) -> Handle:
    if device is None:
        device = torch.cuda.current_device()
    hs = getattr(_tls, "handles", None)
    if hs is None:
        hs = _tls.handles = {}
    if device not in hs:
        hs[device] = Handle(device)
    return hs[device]


def synchronize(device: int | None = None):
    default_handle(device).sync()


def bf16_from_numpy(a, device="cuda") -> torch.Tensor:
    """bf16 bit patterns (numpy uint16) -> torch bf16 tensor on `device`."""
    import numpy as np
    return torch.from_numpy(np.ascontiguousarray(a).view(np.int16)).to(device).view(torch.bfloat16)


def u32_from_numpy(a, device="cuda") -> torch.Tensor:
    """packed uint32 words (numpy) -> torch int32 tensor with the same bits on `device`."""
    import numpy as np
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.uint32).view(np.int32)).to(device)


def bf16_to_numpy(t: torch.Tensor):
    import numpy as np
    return t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16)


def _ptr(t: torch.Tensor | None):
    return None if t is None else C.c_void_p(t.data_ptr())


def _need(t, name, dtypes, device):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if t.device.type != "cuda" or (device is not None and t.device != device):
        raise ValueError(f"{name} must live on {device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} has dtype {t.dtype}, expected one of {dtypes}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


_U32 = (torch.uint32, torch.int32)


def quantized_matmul(x, w, scales, biases=None, transpose=True, group_size=64, bits=4, handle=None):
    """x [..., K] bf16 @ dequant(w)^T -> [..., N] bf16 (mx::quantized_matmul, transpose=True)."""
    if not transpose:
        raise NotImplementedError("transpose=False is not implemented")
    _need(x, "x", (torch.bfloat16,), None)
    dev = x.device
    _need(w, "w", _U32, dev)
    _need(scales, "scales", (torch.bfloat16,), dev)
    if biases is not None:
        _need(biases, "biases", (torch.bfloat16,), dev)
    K = x.shape[-1]
    if w.dim() != 2 or w.shape[1] * 32 // bits != K:
        raise ValueError(f"w of shape {tuple(w.shape)} does not match K={K} at {bits} bits")
    N = w.shape[0]
    if scales.shape != (N, K // group_size) or (biases is not None and biases.shape != scales.shape):
        raise ValueError("scales / biases shape mismatch")
    M = x.numel() // K
    out = torch.empty(*x.shape[:-1], N, dtype=torch.bfloat16, device=dev)
    h = handle or default_handle(dev.index)
    h.bind_stream()
    h.check(h.lib.fm_quantized_matmul(h.h, _ptr(x), M, K, _ptr(w), _ptr(scales), _ptr(biases), N, int(transpose),
                                      group_size, bits, _ptr(out)))
    return out


def linear(x, w, scales, biases=None, group_size=64, bits=4, handle=None):
    """fm_linear: the quantized_matmul of a dense layer (LlamaModel::linear_fast), without
    the routing kernel; x [..., K] bf16 -> [..., N] bf16."""
    _need(x, "x", (torch.bfloat16,), None)
    dev = x.device
    _need(w, "w", _U32, dev)
    _need(scales, "scales", (torch.bfloat16,), dev)
    if biases is not None:
        _need(biases, "biases", (torch.bfloat16,), dev)
    K = x.shape[-1]
    if w.dim() != 2 or w.shape[1] * 32 // bits != K:
        raise ValueError(f"w of shape {tuple(w.shape)} does not match K={K} at {bits} bits")
    N = w.shape[0]
    if scales.shape != (N, K // group_size) or (biases is not None and biases.shape != scales.shape):
        raise ValueError("scales / biases shape mismatch")
    out = torch.empty(*x.shape[:-1], N, dtype=torch.bfloat16, device=dev)
    h = handle or default_handle(dev.index)
    h.bind_stream()
    h.check(h.lib.fm_linear(h.h, _ptr(x), x.numel() // K, K, _ptr(w), _ptr(scales), _ptr(biases), N, group_size,
                            bits, _ptr(out)))
    return out


def gather_qmm(x, w, scales, biases=None, lhs_indices=None, rhs_indices=None, transpose=True, group_size=64,
               bits=4, sorted_indices=False, handle=None):
    """mx::gather_qmm: out[i] = x[lhs(i)] @ dequant(w[rhs[i]])^T, shape batch(idx) + [M, N]."""
    if not transpose:
        raise NotImplementedError("transpose=False is not implemented")
    _need(x, "x", (torch.bfloat16,), None)
    dev = x.device
    _need(w, "w", _U32, dev)
    _need(scales, "scales", (torch.bfloat16,), dev)
    if biases is not None:
        _need(biases, "biases", (torch.bfloat16,), dev)
    if x.dim() < 2 or w.dim() != 3:
        raise ValueError("x must be [..., M, K] and w [E, N, K*bits/32]")
    M, K = x.shape[-2], x.shape[-1]
    E, N = w.shape[0], w.shape[1]
    if w.shape[2] * 32 // bits != K:
        raise ValueError("w does not match K")
    if rhs_indices is None:
        raise ValueError("rhs_indices is required")
    _need(rhs_indices, "rhs_indices", _U32, dev)
    x_batch = tuple(x.shape[:-2])
    xb = 1
    for d in x_batch:
        xb *= d
    if lhs_indices is not None:
        _need(lhs_indices, "lhs_indices", _U32, dev)
        if lhs_indices.shape != rhs_indices.shape:
            raise ValueError("lhs_indices and rhs_indices must have the same shape")
        out_batch = tuple(rhs_indices.shape)
    else:
        out_batch = tuple(torch.broadcast_shapes(x_batch, tuple(rhs_indices.shape)))
        if tuple(rhs_indices.shape) != out_batch:
            raise NotImplementedError("rhs_indices must carry the full broadcast batch shape")
        # x batch index i*xb/B is exact for x batch shapes that broadcast as a prefix
        B = rhs_indices.numel()
        if B % xb:
            raise NotImplementedError("x batch does not broadcast as a prefix of the index batch")
    B = rhs_indices.numel()
    out = torch.empty(*out_batch, M, N, dtype=torch.bfloat16, device=dev)
    h = handle or default_handle(dev.index)
    h.bind_stream()
    h.check(h.lib.fm_gather_qmm(h.h, _ptr(x), xb, M, K, _ptr(w), _ptr(scales), _ptr(biases), E, N,
                                _ptr(lhs_indices), _ptr(rhs_indices), B, int(transpose), group_size, bits,
                                int(sorted_indices), _ptr(out)))
    return out


@dataclass
class MoEWeightsT:
    """Stacked MoE-layer weights as torch CUDA tensors (MoEWeights, model.h:56-72)."""
    router_w: torch.Tensor
    gate: tuple
    up: tuple
    down: tuple
    shared_gate: tuple | None = None
    shared_up: tuple | None = None
    shared_down: tuple | None = None
    shared_expert_gate_w: torch.Tensor | None = None
    router_bias: torch.Tensor | None = None

    @staticmethod
    def from_numpy(d: dict, device) -> "MoEWeightsT":
        def bf(a):
            return bf16_from_numpy(a, device)

        def q(t):
            w, s, b = t
            return (u32_from_numpy(w, device), bf(s), bf(b) if b is not None else None)

        return MoEWeightsT(
            router_w=bf(d["router_w"]), gate=q(d["gate"]), up=q(d["up"]), down=q(d["down"]),
            shared_gate=q(d["shared_gate"]) if "shared_gate" in d else None,
            shared_up=q(d["shared_up"]) if "shared_up" in d else None,
            shared_down=q(d["shared_down"]) if "shared_down" in d else None,
            shared_expert_gate_w=bf(d["shared_expert_gate_w"]) if "shared_expert_gate_w" in d else None,
            router_bias=bf(d["router_bias"]) if "router_bias" in d else None)


def _qw(t):
    if t is None:
        return QWeight(None, None, None)
    w, s, b = t
    return QWeight(w.data_ptr(), s.data_ptr(), b.data_ptr() if b is not None else None)


class MoEBlock:
    """LlamaModel::moe_block on libflashmoe.  cfg: synthetic.MoEShape-like object."""

    def __init__(self, shape, weights: MoEWeightsT, handle: Handle | None = None):
        self.shape = shape
        self.weights = weights
        self.handle = handle
        c = MoEConfig()
        c.hidden, c.inter, c.num_experts, c.top_k = shape.hidden, shape.inter, shape.num_experts, shape.top_k
        c.group_size, c.bits = shape.group_size, shape.bits
        c.norm_topk_prob = int(shape.norm_topk_prob)
        c.shared_inter = shape.shared_inter
        c.router_quantized = 0
        c.shared_gate_quantized = 0
        self.cfg = c
        W = MoEWeights()
        W.router_w = weights.router_w.data_ptr()
        W.gate, W.up, W.down = _qw(weights.gate), _qw(weights.up), _qw(weights.down)
        W.shared_gate, W.shared_up, W.shared_down = (_qw(weights.shared_gate), _qw(weights.shared_up),
                                                     _qw(weights.shared_down))
        if weights.shared_expert_gate_w is not None:
            W.shared_expert_gate_w = weights.shared_expert_gate_w.data_ptr()
        if weights.router_bias is not None:
            W.router_bias = weights.router_bias.data_ptr()
        self.W = W

    def _h(self, device):
        return self.handle or default_handle(device.index)

    def reserve(self, max_tokens: int, device=None):
        h = self._h(device or self.weights.router_w.device)
        h.check(h.lib.fm_reserve(h.h, C.byref(self.cfg), max_tokens))

    def __call__(self, x: torch.Tensor, out: torch.Tensor | None = None, return_routing: bool = False):
        _need(x, "x", (torch.bfloat16,), self.weights.router_w.device)
        if x.shape[-1] != self.shape.hidden:
            raise ValueError("x last dim must equal hidden size")
        T = x.numel() // self.shape.hidden
        y = out if out is not None else torch.empty_like(x)
        outs = MoEOutputs()
        routing = None
        if return_routing:
            k, E = self.shape.top_k, self.shape.num_experts
            routing = {
                "topk_ids": torch.empty(T, k, dtype=torch.int32, device=x.device),
                "topk_scores": torch.empty(T, k, dtype=torch.bfloat16, device=x.device),
                "sorted_token": torch.empty(T * k, dtype=torch.int32, device=x.device),
                "expert_offsets": torch.empty(E + 1, dtype=torch.int32, device=x.device),
            }
            for n, t in routing.items():
                setattr(outs, n, t.data_ptr())
        h = self._h(x.device)
        h.bind_stream()
        h.check(h.lib.fm_moe_block(h.h, C.byref(self.cfg), C.byref(self.W), _ptr(x), T, _ptr(y), C.byref(outs)))
        return (y, routing) if return_routing else y
class MoEBlockVariant:
    """fm_moe_block_variant: the MoE block with another routing / expert form, e.g.
    NemotronHModel::moe_block (server/src/nemotron_h.cpp:1010-1106): sigmoid routing with
    an e_score_correction_bias and group-limited top-k, fp32 scores times
    routed_scaling_factor, ungated relu^2 experts (fc1 as weights.up, fc2 as weights.down)
    and an ungated shared expert (shared_up, shared_down).  Runs the GEMV expert path."""

    def __init__(self, shape, weights: MoEWeightsT, score_func: int = _lib.FM_SCORE_SIGMOID,
                 expert_act: int = _lib.FM_ACT_RELU2, shared_ungated: bool = True, n_group: int = 1,
                 topk_group: int = 1, routed_scaling_factor: float = 1.0,
                 correction_bias: torch.Tensor | None = None, handle: Handle | None = None):
        self.block = MoEBlock(shape, weights, handle)
        self.shape = shape
        if correction_bias is not None:
            _need(correction_bias, "correction_bias", (torch.float32,), weights.router_w.device)
        self.correction_bias = correction_bias
        v = _lib.MoEVariant()
        v.score_func, v.expert_act, v.shared_ungated = score_func, expert_act, int(shared_ungated)
        v.n_group, v.topk_group, v.routed_scaling_factor = n_group, topk_group, routed_scaling_factor
        v.correction_bias = correction_bias.data_ptr() if correction_bias is not None else None
        self.variant = v

    @staticmethod
    def sigmoid_from_numpy(shape, layer: dict, device, n_group: int = 1, topk_group: int = 1,
                           routed_scaling_factor: float = 1.0, handle: Handle | None = None) -> "MoEBlockVariant":
        """The Nemotron-H form from a synthetic.make_sigmoid_layer-style dict."""
        import numpy as np

        def q(t):
            w, sc, b = t
            return (u32_from_numpy(w, device), bf16_from_numpy(sc, device),
                    bf16_from_numpy(b, device) if b is not None else None)
        W = MoEWeightsT(router_w=bf16_from_numpy(layer["router_w"], device), gate=None, up=q(layer["fc1"]),
                        down=q(layer["fc2"]),
                        shared_up=q(layer["shared_up"]) if "shared_up" in layer else None,
                        shared_down=q(layer["shared_down"]) if "shared_down" in layer else None)
        cb = layer.get("correction_bias")
        cbt = torch.from_numpy(np.ascontiguousarray(cb, np.float32)).to(device) if cb is not None else None
        return MoEBlockVariant(shape, W, n_group=n_group, topk_group=topk_group,
                               routed_scaling_factor=routed_scaling_factor, correction_bias=cbt, handle=handle)

    def __call__(self, x: torch.Tensor, out: torch.Tensor | None = None, return_routing: bool = False):
        w = self.block.weights
        _need(x, "x", (torch.bfloat16,), w.router_w.device)
        if x.shape[-1] != self.shape.hidden:
            raise ValueError("x last dim must equal hidden size")
        T = x.numel() // self.shape.hidden
        y = out if out is not None else torch.empty_like(x)
        outs = MoEOutputs()
        routing = None
        self.variant.topk_scores_f32 = None
        if return_routing:
            k = self.shape.top_k
            routing = {"topk_ids": torch.empty(T, k, dtype=torch.int32, device=x.device),
                       "topk_scores_f32": torch.empty(T, k, dtype=torch.float32, device=x.device)}
            outs.topk_ids = routing["topk_ids"].data_ptr()
            self.variant.topk_scores_f32 = routing["topk_scores_f32"].data_ptr()
        h = self.block._h(x.device)
        h.bind_stream()
        h.check(h.lib.fm_moe_block_variant(h.h, C.byref(self.block.cfg), C.byref(self.variant), C.byref(self.block.W),
                                           _ptr(x), T, _ptr(y), C.byref(outs)))
        return (y, routing) if return_routing else y




# ---------------------------------------------------------------- decoder ops
# The rest of the reference's decoder layer (model.cpp:486-656, sampling.cpp:5-7) on the
# same handle and stream as the MoE calls.

def dequantize(w, scales, biases=None, group_size=64, bits=4, handle=None) -> torch.Tensor:
    """mx::dequantize: [N, K*bits/32] codes -> [N, K] bf16 (bf16(fma(s, q, b)))."""
    _need(w, "w", _U32, None)
    dev = w.device
    _need(scales, "scales", (torch.bfloat16,), dev)
    if biases is not None:
        _need(biases, "biases", (torch.bfloat16,), dev)
    N, K = w.shape[0], w.shape[1] * 32 // bits
    if scales.shape != (N, K // group_size) or (biases is not None and biases.shape != scales.shape):
        raise ValueError("scales / biases shape mismatch")
    out = torch.empty(N, K, dtype=torch.bfloat16, device=dev)
    h = handle or default_handle(dev.index)
    h.bind_stream()
    h.check(h.lib.fm_dequantize(h.h, _ptr(w), _ptr(scales), _ptr(biases), N, K, group_size, bits, _ptr(out)))
    return out


def embed(table, ids, handle=None) -> torch.Tensor:
    """mx::take(table, ids, 0): table [V, H] bf16, ids int32 [...] -> [..., H]."""
    _need(table, "table", (torch.bfloat16,), None)
    dev = table.device
    _need(ids, "ids", (torch.int32,), dev)
    V, H = table.shape
    out = torch.empty(*ids.shape, H, dtype=torch.bfloat16, device=dev)
    h = handle or default_handle(dev.index)
    h.bind_stream()
    h.check(h.lib.fm_embed(h.h, _ptr(table), V, H, _ptr(ids), ids.numel(), _ptr(out)))
    return out


def rms_norm(x, weight, eps, residual=None, h_out=None, handle=None) -> torch.Tensor:
    """mx::fast::rms_norm(x + residual, weight, eps) over the last axis; x + residual (bf16)
    is also written to h_out when given (it may be x)."""
    _need(x, "x", (torch.bfloat16,), None)
    dev = x.device
    _need(weight, "weight", (torch.bfloat16,), dev)
    H = x.shape[-1]
    if weight.numel() != H:
        raise ValueError("weight size differs from the last axis")
    for t, n in ((residual, "residual"), (h_out, "h_out")):
        if t is not None:
            _need(t, n, (torch.bfloat16,), dev)
            if t.shape != x.shape:
                raise ValueError(f"{n} shape differs from x")
    y = torch.empty_like(x)
    h = handle or default_handle(dev.index)
    h.bind_stream()
    h.check(h.lib.fm_rms_norm(h.h, _ptr(x), _ptr(residual), _ptr(weight), x.numel() // H, H, float(eps),
                              _ptr(h_out), _ptr(y)))
    return y


def attention(q, k, v, cache_k, cache_v, B, L, offset, rope_theta, q_bias=None, k_bias=None, v_bias=None,
              scale=0.0, q_norm=None, k_norm=None, norm_eps=1e-6, handle=None) -> torch.Tensor:
    """The attention step after the q/k/v projections (model.cpp:560-635): bias adds, the
    optional per-head q / k RMSNorm (QK-norm weights [d]), RoPE at offset + l, k / v into
    the caches [B, n_kv, max_len, d] at [offset, offset+L), causal SDPA.  q [B*L, nh*d] is
    rotated in place; returns [B*L, nh*d] bf16."""
    _need(q, "q", (torch.bfloat16,), None)
    dev = q.device
    for t, n in ((k, "k"), (v, "v"), (cache_k, "cache_k"), (cache_v, "cache_v")):
        _need(t, n, (torch.bfloat16,), dev)
    for t, n in ((q_bias, "q_bias"), (k_bias, "k_bias"), (v_bias, "v_bias"), (q_norm, "q_norm"), (k_norm, "k_norm")):
        if t is not None:
            _need(t, n, (torch.bfloat16,), dev)
    if cache_k.dim() != 4 or cache_v.shape != cache_k.shape or cache_k.shape[0] < B:
        raise ValueError("caches must be [>= B, n_kv, max_len, d] and alike")
    _, nkv, max_len, d = cache_k.shape
    nh = q.shape[-1] // d
    if q.numel() != B * L * nh * d or k.numel() != B * L * nkv * d or v.numel() != k.numel():
        raise ValueError("q / k / v sizes do not match B, L and the cache heads")
    cfg = _lib.AttnConfig(nh, nkv, d, max_len, float(rope_theta), float(scale), float(norm_eps))
    out = torch.empty(B * L, nh * d, dtype=torch.bfloat16, device=dev)
    h = handle or default_handle(dev.index)
    h.bind_stream()
    h.check(h.lib.fm_attention(h.h, C.byref(cfg), _ptr(q), _ptr(k), _ptr(v), _ptr(q_bias), _ptr(k_bias),
                               _ptr(v_bias), _ptr(q_norm), _ptr(k_norm), _ptr(cache_k), _ptr(cache_v), B, L, offset,
                               _ptr(out)))
    return out


def attention_qkv(qkv, cache_k, cache_v, B, L, offset, rope_theta, q_bias=None, k_bias=None, v_bias=None,
                  scale=0.0, q_norm=None, k_norm=None, norm_eps=1e-6, handle=None) -> torch.Tensor:
    """attention() on the output of a fused q|k|v projection: qkv [B*L, (nh + 2 n_kv) * d]
    holds q, k and v side by side in each row (fm_attn_config.qkv_ld); its q columns are
    rotated in place.  Returns [B*L, nh*d] bf16."""
    _need(qkv, "qkv", (torch.bfloat16,), None)
    dev = qkv.device
    for t, n in ((cache_k, "cache_k"), (cache_v, "cache_v")):
        _need(t, n, (torch.bfloat16,), dev)
    for t, n in ((q_bias, "q_bias"), (k_bias, "k_bias"), (v_bias, "v_bias"), (q_norm, "q_norm"), (k_norm, "k_norm")):
        if t is not None:
            _need(t, n, (torch.bfloat16,), dev)
    if cache_k.dim() != 4 or cache_v.shape != cache_k.shape or cache_k.shape[0] < B:
        raise ValueError("caches must be [>= B, n_kv, max_len, d] and alike")
    _, nkv, max_len, d = cache_k.shape
    W = qkv.shape[-1]
    nh = W // d - 2 * nkv
    if qkv.numel() != B * L * W or W % d or nh <= 0:
        raise ValueError("qkv must be [B*L, (n_heads + 2 n_kv) * d]")
    cfg = _lib.AttnConfig(nh, nkv, d, max_len, float(rope_theta), float(scale), float(norm_eps), W)
    out = torch.empty(B * L, nh * d, dtype=torch.bfloat16, device=dev)
    h = handle or default_handle(dev.index)
    h.bind_stream()
    base = qkv.data_ptr()
    h.check(h.lib.fm_attention(h.h, C.byref(cfg), C.c_void_p(base), C.c_void_p(base + 2 * nh * d),
                               C.c_void_p(base + 2 * (nh + nkv) * d), _ptr(q_bias), _ptr(k_bias), _ptr(v_bias),
                               _ptr(q_norm), _ptr(k_norm), _ptr(cache_k), _ptr(cache_v), B, L, offset, _ptr(out)))
    return out


def swiglu(gate, up, handle=None) -> torch.Tensor:
    """The compiled swiglu of model.cpp:14-25 (silu(g) * u, bf16 after every op)."""
    _need(gate, "gate", (torch.bfloat16,), None)
    _need(up, "up", (torch.bfloat16,), gate.device)
    if up.shape != gate.shape:
        raise ValueError("gate and up shapes differ")
    out = torch.empty_like(gate)
    h = handle or default_handle(gate.device.index)
    h.bind_stream()
    h.check(h.lib.fm_swiglu(h.h, _ptr(gate), _ptr(up), gate.numel(), _ptr(out)))
    return out


def argmax(logits, handle=None) -> torch.Tensor:
    """Greedy sampling: the first index of the largest value along the last axis (int32)."""
    _need(logits, "logits", (torch.bfloat16,), None)
    V = logits.shape[-1]
    out = torch.empty(logits.shape[:-1], dtype=torch.int32, device=logits.device)
    h = handle or default_handle(logits.device.index)
    h.bind_stream()
    h.check(h.lib.fm_argmax(h.h, _ptr(logits), logits.numel() // V, V, _ptr(out)))
    return out


# ---------------------------------------------------------------- serving over long and shared caches

_BF16, _I32, _F32 = (torch.bfloat16,), (torch.int32,), (torch.float32,)
_BF = torch.bfloat16
_ROPE_SCALINGS = {"linear": _lib.FM_ROPE_LINEAR, "ntk": _lib.FM_ROPE_NTK, "yarn": _lib.FM_ROPE_YARN,
                  "banded": _lib.FM_ROPE_BANDED}


@functools.lru_cache(maxsize=256)
def _rope_config_of(d, theta, rotary_dim, traditional, scaling) -> _lib.RopeConfig:
    c = _lib.RopeConfig(d, rotary_dim or 0, int(traditional), _lib.FM_ROPE_UNSCALED, theta)
    if rotary_dim is not None and not 0 < rotary_dim <= d:
        raise ValueError("rotary_dim must be between 2 and the head size")
    if scaling is not None:
        s = dict(scaling)
        kind = s.pop("type", None)
        if kind not in _ROPE_SCALINGS:
            raise ValueError(f"unknown rope scaling {kind!r}, expected one of {sorted(_ROPE_SCALINGS)}")
        c.scaling, c.factor = _ROPE_SCALINGS[kind], float(s.pop("factor"))
        c.attn_factor = float(s.pop("attn_factor", 0.0))
        if kind in ("yarn", "banded"):
            lo, hi = ("beta_slow", "beta_fast") if kind == "yarn" else ("low_freq", "high_freq")
            c.original_len = float(s.pop("original_len"))
            c.low, c.high = float(s.pop(lo, 1.0)), float(s.pop(hi, 32.0 if kind == "yarn" else 4.0))
        if s:
            raise ValueError(f"unknown {kind} scaling entries {sorted(s)}")
    return c


def _rope_config(d, theta, rotary_dim, traditional, scaling) -> _lib.RopeConfig:
    return _rope_config_of(d, float(theta), rotary_dim, bool(traditional),
                           None if scaling is None else tuple(sorted(scaling.items())))


def _heads_ld(t, name, index, shape, step):
    """Checks [..., heads, d] bf16 on CUDA device `index` whose heads lie side by side in each token's
    row (`shape` and `step` are t's sizes and strides); returns the elements from one token's row
    to the next (leading axes must be one stride apart, in order)."""
    if t.get_device() != index:
        raise ValueError(f"{name} must live on CUDA device {index}")
    if t.dtype is not _BF:
        raise ValueError(f"{name} has dtype {t.dtype}, expected torch.bfloat16")
    n = len(shape)
    if n < 3:
        raise ValueError(f"{name} must be [..., heads, head size]")
    h, d = shape[-2], shape[-1]
    if (d > 1 and step[-1] != 1) or (h > 1 and step[-2] != d):
        if t.numel():
            raise ValueError(f"the heads of {name} must lie side by side")
    if n == 3 and shape[0] > 1 and step[0] >= h * d:
        return step[0]
    ld, many = None, 1
    for i in range(n - 3, -1, -1):
        if shape[i] > 1:
            if ld is None:
                ld = step[i]
            elif step[i] != ld * many and t.numel():
                raise ValueError(f"the tokens of {name} must be one stride apart")
            many *= shape[i]
    if ld is None:
        return h * d
    if ld < h * d and t.numel():
        raise ValueError(f"the tokens of {name} may not share memory")
    return ld


def _cuda_index(t, name):
    """The CUDA device a tensor is on."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    index = t.get_device() if t.is_cuda else -1
    if index < 0:
        raise ValueError(f"{name} must live on a CUDA device")
    return index


def _int32(value, name):
    """A Python integer that a C int holds (ctypes would cut it)."""
    value = int(value)
    if not -2 ** 31 <= value < 2 ** 31:
        raise ValueError(f"{name} does not fit 32 bits")
    return value


def _packed(t, name, dtype, index):
    """A contiguous tensor of `dtype` on CUDA device `index`: its data pointer."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != index or not t.is_contiguous():
        _need(t, name, (dtype,), torch.device("cuda", index))
    return t.data_ptr()


def _bound(handle, index):
    """The handle of a call on CUDA device `index`, bound to torch's current stream there."""
    if handle is None:
        handle = default_handle(index)
    elif handle.device != index:
        raise ValueError(f"the handle is of CUDA device {handle.device}, the tensors are on {index}")
    handle.bind_current()
    return handle


def rope(x, positions, theta, rotary_dim=None, traditional=False, scaling=None, out=None, handle=None) -> torch.Tensor:
    """Rotary positions (mx::fast::rope with one position per token): x [..., heads, d] bf16,
    positions int32 [...] (any int32; negative ones rotate back) -> x rotated, in `out` if given
    (it may be x).  rotary_dim leading elements of a head rotate (default all), in pairs
    (i, i + rotary_dim / 2) or, traditional, (2i, 2i + 1).  scaling: None or a dict with
    "type" and "factor": "linear", "ntk", "yarn" (original_len, beta_slow, beta_fast) or
    "banded" (original_len, low_freq, high_freq), and optionally attn_factor.  x and out may
    be views of wider rows (a fused projection's)."""
    dev = _cuda_index(x, "x")
    shape = x.shape
    ld = _heads_ld(x, "x", dev, shape, x.stride())
    pos = _packed(positions, "positions", torch.int32, dev)
    if positions.shape != shape[:-2]:
        raise ValueError("positions must have x's shape without heads and head size")
    cfg = _rope_config(shape[-1], theta, rotary_dim, traditional, scaling)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        out_ld = shape[-2] * shape[-1]
    else:
        _cuda_index(out, "out")
        out_ld = _heads_ld(out, "out", dev, out.shape, out.stride())
        if out.shape != shape:
            raise ValueError("out has another shape than x")
    h = _bound(handle, dev)
    st = h.lib.fm_rope(h.h, cfg, x.data_ptr(), ld, shape[-2], pos, positions.numel(), out.data_ptr(), out_ld)
    if st:
        h.check(st)
    return out


def rope_append(q, k, v, positions, slots, cache_k, cache_v, theta, traditional=False, scaling=None, rotary_dim=None,
                out=None, handle=None) -> torch.Tensor:
    """A step's q [T, nh, d], k and v [T, n_kv, d] (views of a fused projection's rows, or
    separate) with T = B * L tokens in sequence order: returns q rotated at positions [T] (in
    `out` if given, which may be q); k rotated and v go into the caches [B, n_kv, max_len, d]
    at slots [T] (a negative slot writes nothing; a sequence's slots must differ)."""
    dev = _cuda_index(q, "q")
    if not (isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor)):
        raise TypeError("k and v must be torch tensors")
    q_shape, k_shape, c_shape = q.shape, k.shape, cache_k.shape
    ld = _heads_ld(q, "q", dev, q_shape, q.stride())
    kv_ld = _heads_ld(k, "k", dev, k_shape, k.stride())
    if _heads_ld(v, "v", dev, v.shape, v.stride()) != kv_ld or v.shape != k_shape:
        raise ValueError("k and v must have the same shape and strides")
    ck, cv = _packed(cache_k, "cache_k", _BF, dev), _packed(cache_v, "cache_v", _BF, dev)
    pos, slot = _packed(positions, "positions", torch.int32, dev), _packed(slots, "slots", torch.int32, dev)
    T, nh, d = positions.numel(), q_shape[-2], q_shape[-1]
    if len(c_shape) != 4 or cache_v.shape != c_shape or c_shape[3] != d or k_shape[-1] != d or k_shape[-2] != c_shape[1]:
        raise ValueError("caches must be [B, n_kv, max_len, d] with k's heads and q's head size")
    B = c_shape[0]
    if T % max(B, 1) or (B == 0 and T) or slots.numel() != T or q.numel() != T * nh * d or k.numel() != T * k_shape[-2] * d:
        raise ValueError("q, k, v, positions and slots must hold the same T = B * L tokens")
    cfg = _rope_config(d, theta, rotary_dim, traditional, scaling)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        out_ld = nh * d
    else:
        _cuda_index(out, "out")
        out_ld = _heads_ld(out, "out", dev, out.shape, out.stride())
        if out.shape != q_shape:
            raise ValueError("out has another shape than q")
    h = _bound(handle, dev)
    st = h.lib.fm_rope_append(h.h, cfg, q.data_ptr(), ld, nh, k.data_ptr(), v.data_ptr(), kv_ld, k_shape[-2], pos, slot, B,
                              T // max(B, 1), ck, cv, c_shape[2], out.data_ptr(), out_ld)
    if st:
        h.check(st)
    return out


def _cache_attn(q, prefix_k, prefix_v, prefix_len, cache_k, cache_v, lens, acc, scale, handle):
    dev = _cuda_index(q, "q")
    q_shape = q.shape
    ld = _heads_ld(q, "q", dev, q_shape, q.stride())
    if len(q_shape) != 4:
        raise ValueError("q must be [B, L, n_heads, d]")
    B, L, nh, d = q_shape
    nkv = max_len = prefix_max = 0
    pk = pv = ck = cv = n = None
    if cache_k is not None:
        ck, cv = _packed(cache_k, "cache_k", _BF, dev), _packed(cache_v, "cache_v", _BF, dev)
        shape = cache_k.shape
        if len(shape) != 4 or shape[0] != B or shape[3] != d or cache_v.shape != shape:
            raise ValueError("caches must be [B, n_kv, max_len, d] with q's batch and head size, and alike")
        nkv, max_len = shape[1], shape[2]
        if lens is None:
            raise ValueError("lens is required with caches")
        n = _packed(lens, "lens", torch.int32, dev)
        if lens.shape != (B,):
            raise ValueError("lens must be [B]")
    elif lens is not None or prefix_k is None:
        raise ValueError("caches (or a prefix, without lens) are needed")
    if prefix_k is not None:
        pk, pv = _packed(prefix_k, "prefix_k", _BF, dev), _packed(prefix_v, "prefix_v", _BF, dev)
        shape = prefix_k.shape
        if len(shape) != 3 or shape[2] != d or prefix_v.shape != shape or (cache_k is not None and shape[0] != nkv):
            raise ValueError("the prefix must be [n_kv, length, d] with the caches' heads and q's head size, k and v alike")
        nkv, prefix_max = shape[0], shape[1]
        prefix_len = prefix_max if prefix_len is None else int(prefix_len)
        if not 0 <= prefix_len <= prefix_max:
            raise ValueError("prefix_len is not within the prefix")
    if nkv == 0 or nh % nkv:
        raise ValueError("n_heads must be a multiple of n_kv")
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    cfg = _lib.CacheAttnConfig(nh, nkv, d, max_len, prefix_max, _int32(ld, "q's stride"), scale)
    if cfg.scale == 0.0 != scale:
        raise ValueError("scale is too small")
    h = _bound(handle, dev)
    if acc is None:
        st = h.lib.fm_attention_prefix(h.h, cfg, q.data_ptr(), pk, pv, prefix_len or 0, ck, cv, n, B, L, out.data_ptr())
    else:
        a = _packed(acc, "acc", torch.float32, dev)
        if acc.shape != cache_k.shape[:3]:
            raise ValueError("acc must be [B, n_kv, max_len]")
        st = h.lib.fm_attention_scored(h.h, cfg, q.data_ptr(), ck, cv, n, B, L, a, out.data_ptr())
    if st:
        h.check(st)
    return out


def attention_prefix(q, prefix_k, prefix_v, cache_k=None, cache_v=None, lens=None, prefix_len=None, scale=0.0,
                     handle=None) -> torch.Tensor:
    """Attention of a batch whose sequences share a prefix, read once for all: q [B, L, nh, d]
    (rotated; a view of wider rows may be given), prefix_k / prefix_v [n_kv, P, d] of which the
    first prefix_len rows count (default all), and each sequence's own caches
    [B, n_kv, max_len, d] with lens [B] int32 filled slots, the L new tokens' among them:
    token l sees the prefix and the slots j <= lens[b] - L + l.  scale 0: 1/sqrt(d).  Returns
    [B, L, nh, d].  Calls of one handle (the thread's default one without `handle`) on several
    streams wait for one another; those that are to overlap, and replays of captured calls that
    may, need a handle each."""
    return _cache_attn(q, prefix_k, prefix_v, prefix_len, cache_k, cache_v, lens, None, scale, handle)


def attention_scored(q, cache_k, cache_v, lens, acc, scale=0.0, handle=None) -> torch.Tensor:
    """attention_prefix without a prefix that also adds to acc [B, n_kv, max_len] fp32 each
    slot's attention probabilities, summed over the kv head's query heads and the L tokens.
    Streams and handles as for attention_prefix."""
    if acc is None:
        raise TypeError("acc must be a torch tensor")
    return _cache_attn(q, None, None, None, cache_k, cache_v, lens, acc, scale, handle)


def cache_evict(cache_k, cache_v, acc, lens, budget, sinks=0, recent=0, positions=None, out=None, lens_out=None,
                handle=None) -> torch.Tensor:
    """Cuts every (sequence, kv head) of the caches [B, n_kv, max_len, d] down to
    n = min(lens[b], budget) slots, those of the largest acc [B, n_kv, max_len]; positions
    below `sinks` and above the newest - `recent` stay whatever their weight (positions
    [B, n_kv, max_len] int32, a slot's index without them).  In place, or into
    out = (k, v, acc, positions) of [B, n_kv, M >= budget, ...] (positions may be None when
    `positions` is).  Slots that stay below n keep their places, the others below n take those
    from n on in order.  Returns the new lengths [B] (lens_out if given; it may be lens).
    Streams and handles as for attention_prefix."""
    dev = _cuda_index(cache_k, "cache_k")
    shape = cache_k.shape
    ck, cv = _packed(cache_k, "cache_k", _BF, dev), _packed(cache_v, "cache_v", _BF, dev)
    if len(shape) != 4 or cache_v.shape != shape:
        raise ValueError("caches must be [B, n_kv, max_len, d] and alike")
    B, nkv, max_len, d = shape
    a = _packed(acc, "acc", torch.float32, dev)
    p = None if positions is None else _packed(positions, "positions", torch.int32, dev)
    if acc.shape != shape[:3] or (positions is not None and positions.shape != shape[:3]):
        raise ValueError("acc and positions must be [B, n_kv, max_len]")
    if out is None:
        rows, ok, ov, oa, op = max_len, ck, cv, a, p
    else:
        out_k, out_v, out_acc, out_positions = out
        ok, ov = _packed(out_k, "out k", _BF, dev), _packed(out_v, "out v", _BF, dev)
        oa = _packed(out_acc, "out acc", torch.float32, dev)
        op = None if out_positions is None else _packed(out_positions, "out positions", torch.int32, dev)
        rows = out_k.shape[2] if out_k.dim() == 4 else -1
        if out_k.shape != (B, nkv, rows, d) or out_v.shape != out_k.shape or out_acc.shape != (B, nkv, rows) or \
                (out_positions is not None and out_positions.shape != (B, nkv, rows)):
            raise ValueError("the outputs must be [B, n_kv, length, d] (k, v) and [B, n_kv, length] (acc, positions)")
    n = _packed(lens, "lens", torch.int32, dev)
    if lens_out is None:
        lens_out = torch.empty_like(lens)
    no = _packed(lens_out, "lens_out", torch.int32, dev)
    if lens.shape != (B,) or lens_out.shape != (B,):
        raise ValueError("lens and lens_out must be [B]")
    cfg = _lib.EvictConfig(nkv, d, max_len, rows, _int32(budget, "budget"), _int32(sinks, "sinks"), _int32(recent, "recent"))
    h = _bound(handle, dev)
    st = h.lib.fm_cache_evict(h.h, cfg, ck, cv, a, p, n, B, ok, ov, oa, op, no)
    if st:
        h.check(st)
    return lens_out
