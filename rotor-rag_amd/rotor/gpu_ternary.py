"""HIP backend of the ternary linear for MI355X (gfx950).

Drop-in for the reference's OpenCL plug-in ``GPUTernaryOps``
(src/rotor/gpu_ternary.py:73-208): same duck type -- ``pack_ternary_weights(W)`` and
``ternary_matmul(packed, scales, input_vec, in_dim, out_dim)`` -- plus batched entry
points (``linear``, ``linear_i32``, ``quantize_rows``, ``plan``) that the reference
lacks (it loops over tokens, src/rotor/transformer.py:134-143).

Differences from the reference, by design:
  * weights are uploaded once and stay resident (the reference re-uploads them on
    every call, src/rotor/gpu_ternary.py:160-164);
  * activations are quantised per token to int8 (absmax, src/rotor/quantization.py:
    137-149 per row) and accumulated exactly in int32 (W2A8);
  * any failure raises ``RuntimeError``; nothing falls back to the CPU.

PyTorch supplies device memory and the stream; the compute is the HIP library.
"""
from __future__ import annotations

import ctypes
import functools
import operator

import numpy as np

from . import _hip
from .format import pack_rotor_rows, unpack_rotor_rows


def _torch():
    import torch

    return torch


@functools.lru_cache(maxsize=1024)
def _kv4_workspace_bytes(B, M, H, Hkv, hd, Lmax):
    return _hip.load().rt_kv4_attention_workspace(B, M, H, Hkv, hd, Lmax)


@functools.lru_cache(maxsize=1024)
def _paged_workspace_bytes(kind, Hkv, page, hd, B, P, H, weights):
    rows = Hkv * page * hd
    return _hip.load().rt_paged_attention_workspace(_hip.PAGES.pack(16, rows, rows, 16, 16, kind, 1, Hkv, page, hd, B, P), H, weights)


@functools.lru_cache(maxsize=1024)
def _paged_evict_workspace_bytes(kind, Hkv, page, hd, B, P):
    rows = Hkv * page * hd
    return _hip.load().rt_paged_evict_workspace(_hip.PAGES.pack(16, rows, rows, 16, 16, kind, 1, Hkv, page, hd, B, P))


@functools.lru_cache(maxsize=1)
def _paged_types():
    torch = _torch()
    return {torch.float32: _hip.PAGED_F32, torch.bfloat16: _hip.PAGED_BF16, torch.float16: _hip.PAGED_F16}


class DeviceTernaryWeights:
    """A device-resident ternary matrix (opaque ``rt_weights`` handle)."""

    def __init__(self, backend: "HIPTernaryOps", handle: ctypes.c_void_p, N: int, K: int, scale: float):
        self._backend = backend
        self.handle = handle
        self.out_features = N
        self.in_features = K
        self.scale = float(scale)

    @property
    def shape(self):
        return (self.out_features, self.in_features)

    def download(self) -> np.ndarray:
        """Rotor bytes [N, ceil(K/4)] read back from the device (inverse of the upload)."""
        out = np.empty((self.out_features, (self.in_features + 3) // 4), dtype=np.uint8)
        lib = _hip.load()
        _hip.check(lib.rt_weights_download(self._backend.ctx, self.handle, out.ctypes.data), "rt_weights_download")
        return out

    def free(self) -> None:
        if self.handle:
            _hip.load().rt_weights_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class LinearPlan:
    """G ternary linears prepared for one launch (see rt_plan_create)."""

    def __init__(self, backend, handle, keep):
        self._backend = backend
        self.handle = handle
        self._keep = keep  # tensors / weights the plan's device pointers refer to

    def run(self) -> None:
        """Run the plan: one launch at M = 1 when the GEMV quantises in its prologue,
        else quantize() then gemv()."""
        b = self._backend
        b._bind_stream()
        _hip.check(_hip.load().rt_plan_run(b.ctx, self.handle), "rt_plan_run")

    def quantize(self) -> None:
        """Two-launch form of run(), first launch: per-token quantisation of the distinct inputs."""
        b = self._backend
        b._bind_stream()
        _hip.check(_hip.load().rt_plan_quantize(b.ctx, self.handle), "rt_plan_quantize")

    def gemv(self) -> None:
        """Two-launch form of run(), second launch: the ternary GEMV over all problems."""
        b = self._backend
        b._bind_stream()
        _hip.check(_hip.load().rt_plan_gemv(b.ctx, self.handle), "rt_plan_gemv")

    def attach_attention(self, k_cache, v_cache, rope, H: int, Hkv: int, hd: int, Lmax: int, pos, workspace) -> None:
        """Run the decode RoPE + KV append + attention partials of the token inside run()'s
        launch of this q/k/v plan (rt_plan_attach_attention; the arguments of
        rt_rope_attention_decode).  k_cache=None detaches."""
        if k_cache is None:
            _hip.check(_hip.load().rt_plan_attach_attention(self.handle, None, None, None, 0, 0, 0, 0, None, None, 0),
                       "rt_plan_attach_attention")
            return
        _hip.check(_hip.load().rt_plan_attach_attention(self.handle, k_cache.data_ptr(), v_cache.data_ptr(),
                                                        rope.data_ptr(), H, Hkv, hd, Lmax, pos.data_ptr(),
                                                        workspace.data_ptr(), workspace.numel() * workspace.element_size()),
                   "rt_plan_attach_attention")
        self._keep = (self._keep, k_cache, v_cache, rope, pos, workspace)

    def attention_combine(self, out, ssq) -> None:
        """Also combine the attention partials in run()'s launch (rt_plan_attention_combine):
        out fp32 [H*hd] receives the attention output, ssq float64 [H*hd/32] the sums of its
        squares per 32 outputs (an SRC_RMSNORM_SSQ plan's x and aux2).  (None, None) detaches."""
        if (out is None) != (ssq is None):
            raise ValueError("attention_combine: give both out and ssq, or neither")
        if out is not None:
            torch = _torch()
            if (out.dtype != torch.float32 or ssq.dtype != torch.float64 or not out.is_contiguous()
                    or not ssq.is_contiguous() or ssq.numel() * 32 < out.numel()):
                raise ValueError("attention_combine: out float32 [H*hd], ssq float64 [H*hd/32], contiguous")
        ptr = lambda t: t.data_ptr() if t is not None else None
        _hip.check(_hip.load().rt_plan_attention_combine(self.handle, ptr(out), ptr(ssq)), "rt_plan_attention_combine")
        self._keep = (self._keep, out, ssq)

    def set_output_ssq(self, ssq) -> None:
        """Also write, per 32 outputs (after the residual), the float64 sum of their squares
        into ssq [ceil(N/32)] (rt_plan_set_output_ssq; one-problem fused decode plans): the
        aux2 of an SRC_RMSNORM_SSQ plan reading this plan's output.  None detaches."""
        if ssq is not None:
            torch = _torch()
            if ssq.dtype != torch.float64 or not ssq.is_contiguous():
                raise ValueError("set_output_ssq: ssq float64, contiguous")
        _hip.check(_hip.load().rt_plan_set_output_ssq(self.handle, ssq.data_ptr() if ssq is not None else None),
                   "rt_plan_set_output_ssq")
        self._keep = (self._keep, ssq)

    def attention_timeouts(self) -> int:
        """Attention waits of this plan's launches that gave up (rt_plan_attention_timeouts;
        synchronises the device).  Never expected: a non-zero count means wrong results."""
        n = ctypes.c_int()
        _hip.check(_hip.load().rt_plan_attention_timeouts(self.handle, ctypes.byref(n)), "rt_plan_attention_timeouts")
        return n.value

    def describe(self):
        """(kind, tile_m, tile_n, workgroups) of the launch the plan makes (rt_plan_describe);
        kind is one of _hip.LAUNCH_*."""
        v = [ctypes.c_int() for _ in range(4)]
        _hip.check(_hip.load().rt_plan_describe(self.handle, *[ctypes.byref(x) for x in v]), "rt_plan_describe")
        return tuple(x.value for x in v)

    def free(self) -> None:
        if self.handle:
            _hip.load().rt_plan_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class DeviceActivations:
    """Reusable quantised activations (opaque ``rt_act``): up to ``capacity`` tokens of
    ``in_features`` int8 values in the device layout, plus per-token scales."""

    def __init__(self, backend, handle, capacity: int, K: int):
        self._backend = backend
        self.handle = handle
        self.capacity = capacity
        self.in_features = K
        self.tokens = 0

    def export(self):
        """(q int8 [M, K], s fp32 [M]) device tensors of the tokens held, natural order."""
        torch = _torch()
        b = self._backend
        q = torch.empty((self.tokens, self.in_features), dtype=torch.int8, device=b.device)
        s = torch.empty((self.tokens,), dtype=torch.float32, device=b.device)
        b._bind_stream()
        _hip.check(_hip.load().rt_act_export(b.ctx, self.handle, q.data_ptr(), s.data_ptr()), "rt_act_export")
        return q, s

    def free(self) -> None:
        if self.handle:
            _hip.load().rt_act_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class HIPTernaryOps:
    """GPUTernaryOps-compatible HIP backend bound to one device."""

    def __init__(self, device: int = 0):
        torch = _torch()
        self.lib = _hip.load()
        if not torch.cuda.is_available():
            raise RuntimeError("HIPTernaryOps: no GPU visible to PyTorch-ROCm")
        self.device_index = int(device)
        self.device = torch.device("cuda", self.device_index)
        ctx = ctypes.c_void_p()
        _hip.check(self.lib.rt_ctx_create(self.device_index, ctypes.byref(ctx)), "rt_ctx_create")
        self.ctx = ctx
        self._bind_stream()

    # -- plumbing -----------------------------------------------------------------
    def _bind_stream(self):
        torch = _torch()
        s = torch.cuda.current_stream(self.device)
        _hip.check(self.lib.rt_ctx_set_stream(self.ctx, ctypes.c_void_p(s.cuda_stream)), "rt_ctx_set_stream")

    def _dev(self, a, dtype):
        """numpy/torch -> contiguous device tensor of `dtype` on this device."""
        torch = _torch()
        if isinstance(a, torch.Tensor):
            t = a.to(device=self.device, dtype=dtype)
        else:
            t = torch.from_numpy(np.ascontiguousarray(a)).to(device=self.device, dtype=dtype)
        return t.contiguous()

    def synchronize(self):
        _hip.check(self.lib.rt_sync(self.ctx), "rt_sync")

    # -- weights ------------------------------------------------------------------
    def upload(self, rotor_bytes, in_features: int, scale: float = 1.0) -> DeviceTernaryWeights:
        """Rotor bytes [N, ceil(K/4)] (host) -> device-resident weights."""
        p = np.ascontiguousarray(rotor_bytes, dtype=np.uint8)
        if p.ndim != 2 or p.shape[1] != (in_features + 3) // 4:
            raise ValueError(f"rotor bytes of shape {p.shape} do not hold rows of {in_features} weights")
        h = ctypes.c_void_p()
        _hip.check(self.lib.rt_weights_upload(self.ctx, p.ctypes.data, p.shape[0], int(in_features),
                                              float(scale), ctypes.byref(h)), "rt_weights_upload")
        return DeviceTernaryWeights(self, h, p.shape[0], int(in_features), scale)

    def upload_device(self, rotor_bytes_dev, in_features: int, scale: float = 1.0) -> DeviceTernaryWeights:
        """Rotor bytes already on the device (uint8 tensor [N, ceil(K/4)])."""
        t = self._dev(rotor_bytes_dev, _torch().uint8)
        if t.ndim != 2 or t.shape[1] != (in_features + 3) // 4:
            raise ValueError(f"rotor bytes of shape {tuple(t.shape)} do not hold rows of {in_features} weights")
        self._bind_stream()
        h = ctypes.c_void_p()
        _hip.check(self.lib.rt_weights_upload_device(self.ctx, t.data_ptr(), t.shape[0], int(in_features),
                                                     float(scale), ctypes.byref(h)), "rt_weights_upload_device")
        self.synchronize()
        return DeviceTernaryWeights(self, h, t.shape[0], int(in_features), scale)

    def pack_ternary_weights(self, weights, scale: float = 1.0) -> DeviceTernaryWeights:
        """{-1,0,+1} [N, K] -> device weights.  src/rotor/gpu_ternary.py:112-136 (which
        returned host bytes in a w+1 code); here the rotor code is uploaded once."""
        W = np.asarray(weights)
        if W.ndim != 2:
            raise ValueError("pack_ternary_weights expects a 2-D [out, in] matrix")
        return self.upload(pack_rotor_rows(W), W.shape[1], scale)

    # -- compute ------------------------------------------------------------------
    def quantize_rows(self, x):
        """Per-token absmax int8: x [M, K] -> (q int8 [M, K], s fp32 [M]) device tensors."""
        torch = _torch()
        xt = self._dev(x, torch.float32)
        M, K = xt.shape
        q = torch.empty((M, K), dtype=torch.int8, device=self.device)
        s = torch.empty((M,), dtype=torch.float32, device=self.device)
        self._bind_stream()
        _hip.check(self.lib.rt_quantize_rows(self.ctx, xt.data_ptr(), M, K, q.data_ptr(), s.data_ptr()),
                   "rt_quantize_rows")
        return q, s

    def linear_i32(self, w: DeviceTernaryWeights, q):
        """Exact int32 accumulators q [M, K] int8 x W^T -> [M, N] (device tensor)."""
        torch = _torch()
        qt = self._dev(q, torch.int8)
        if qt.ndim != 2 or qt.shape[1] != w.in_features:
            raise ValueError(f"q of shape {tuple(qt.shape)} does not match K={w.in_features}")
        acc = torch.empty((qt.shape[0], w.out_features), dtype=torch.int32, device=self.device)
        self._bind_stream()
        _hip.check(self.lib.rt_linear_i32(self.ctx, w.handle, qt.data_ptr(), qt.shape[0], acc.data_ptr()),
                   "rt_linear_i32")
        return acc

    def linear_device(self, w: DeviceTernaryWeights, x, row_scale=None, out=None):
        """W2A8 ternary linear on device tensors: x [M, K] fp32 -> y [M, N] fp32."""
        torch = _torch()
        xt = self._dev(x, torch.float32)
        if xt.ndim != 2 or xt.shape[1] != w.in_features:
            raise ValueError(f"x of shape {tuple(xt.shape)} does not match K={w.in_features}")
        M = xt.shape[0]
        y = out if out is not None else torch.empty((M, w.out_features), dtype=torch.float32, device=self.device)
        self._bind_stream()
        if row_scale is None:
            _hip.check(self.lib.rt_linear_f32(self.ctx, w.handle, xt.data_ptr(), M, y.data_ptr()), "rt_linear_f32")
        else:
            rs = self._dev(row_scale, torch.float32).reshape(-1)
            if rs.numel() != w.out_features:
                raise ValueError("row scales must have out_features entries")
            _hip.check(self.lib.rt_linear_f32_rowscale(self.ctx, w.handle, xt.data_ptr(), M, rs.data_ptr(),
                                                       y.data_ptr()), "rt_linear_f32_rowscale")
        return y

    def linear(self, w: DeviceTernaryWeights, x):
        """x [M, K] numpy -> numpy y [M, N]; torch in -> torch (device) out."""
        torch = _torch()
        y = self.linear_device(w, x)
        if isinstance(x, torch.Tensor):
            return y
        return y.cpu().numpy()

    def ternary_matmul(self, packed_weights, scales, input_vec, in_dim: int, out_dim: int) -> np.ndarray:
        """Reference duck type (src/rotor/gpu_ternary.py:138-202): one token, per-row
        scales, numpy in and out.  ``packed_weights`` is what pack_ternary_weights
        returned."""
        if not isinstance(packed_weights, DeviceTernaryWeights):
            raise TypeError("packed_weights must come from HIPTernaryOps.pack_ternary_weights")
        if packed_weights.shape != (out_dim, in_dim):
            raise ValueError(f"weights are {packed_weights.shape}, call asked for ({out_dim}, {in_dim})")
        x = np.asarray(input_vec, dtype=np.float32).reshape(1, in_dim)
        y = self.linear_device(packed_weights, x, row_scale=np.asarray(scales, dtype=np.float32))
        return y.cpu().numpy().reshape(out_dim)

    def plan(self, weights, xs, ys) -> LinearPlan:
        """Prepare one launch of len(weights) linears: ys[g] = W_g(xs[g]); device tensors,
        all xs with the same number of rows.  Equal xs tensors share one quantisation."""
        G = len(weights)
        if not (G == len(xs) == len(ys)) or G == 0:
            raise ValueError("plan needs equal, non-zero numbers of weights, inputs and outputs")
        M = xs[0].shape[0]
        for w, x, y in zip(weights, xs, ys):
            if x.shape != (M, w.in_features) or y.shape != (M, w.out_features):
                raise ValueError("plan: tensor shapes do not match the weights")
            if not (x.is_contiguous() and y.is_contiguous()) or x.device != self.device or y.device != self.device:
                raise ValueError("plan: tensors must be contiguous and on the backend's device")
        P = ctypes.c_void_p
        wa = (P * G)(*[w.handle for w in weights])
        xa = (P * G)(*[x.data_ptr() for x in xs])
        ya = (P * G)(*[y.data_ptr() for y in ys])
        h = ctypes.c_void_p()
        _hip.check(self.lib.rt_plan_create(self.ctx, G, wa, xa, M, ya, ctypes.byref(h)), "rt_plan_create")
        return LinearPlan(self, h, (list(weights), list(xs), list(ys)))

    # -- reusable quantised activations ------------------------------------------
    def activations(self, capacity: int, in_features: int) -> DeviceActivations:
        h = ctypes.c_void_p()
        _hip.check(self.lib.rt_act_create(self.ctx, int(capacity), int(in_features), ctypes.byref(h)), "rt_act_create")
        return DeviceActivations(self, h, int(capacity), int(in_features))

    def _check_rows(self, t, act, name):
        if t.ndim != 2 or t.shape[1] != act.in_features or t.shape[0] > act.capacity:
            raise ValueError(f"{name} of shape {tuple(t.shape)} does not fit activations "
                             f"[{act.capacity}, {act.in_features}]")

    def act_quantize(self, x, act: DeviceActivations):
        """act <- per-token int8 of x [M, K] (device)."""
        xt = self._dev(x, _torch().float32)
        self._check_rows(xt, act, "x")
        self._bind_stream()
        _hip.check(self.lib.rt_act_quantize(self.ctx, xt.data_ptr(), xt.shape[0], act.handle), "rt_act_quantize")
        act.tokens = xt.shape[0]
        return act

    def act_rmsnorm_quantize(self, x, norm_w, act: DeviceActivations, eps: float = 1e-6, h_out=None):
        """act <- int8 of RMSNorm(x) * norm_w (fused); optional fp32 h_out [M, K]."""
        torch = _torch()
        xt = self._dev(x, torch.float32)
        wt = self._dev(norm_w, torch.float32).reshape(-1)
        self._check_rows(xt, act, "x")
        if wt.numel() != act.in_features:
            raise ValueError("norm weight must have in_features entries")
        self._bind_stream()
        _hip.check(self.lib.rt_act_rmsnorm_quantize(self.ctx, xt.data_ptr(), wt.data_ptr(), float(eps), xt.shape[0],
                                                    act.handle, h_out.data_ptr() if h_out is not None else None),
                   "rt_act_rmsnorm_quantize")
        act.tokens = xt.shape[0]
        return act

    def act_relu2_mul_quantize(self, gate, up, act: DeviceActivations, a_out=None):
        """act <- int8 of relu(gate)^2 * up (fused); optional fp32 a_out [M, K]."""
        torch = _torch()
        g = self._dev(gate, torch.float32)
        u = self._dev(up, torch.float32)
        self._check_rows(g, act, "gate")
        if u.shape != g.shape:
            raise ValueError("gate and up must have the same shape")
        self._bind_stream()
        _hip.check(self.lib.rt_act_relu2_mul_quantize(self.ctx, g.data_ptr(), u.data_ptr(), g.shape[0], act.handle,
                                                      a_out.data_ptr() if a_out is not None else None),
                   "rt_act_relu2_mul_quantize")
        act.tokens = g.shape[0]
        return act

    def act_relu2_mul_norm_quantize(self, gate, up, norm_w, act: DeviceActivations, eps: float = 1e-6, a_out=None):
        """act <- int8 of RMSNorm(relu(gate)^2 * up) * norm_w (fused)."""
        torch = _torch()
        g = self._dev(gate, torch.float32)
        u = self._dev(up, torch.float32)
        wt = self._dev(norm_w, torch.float32).reshape(-1)
        self._check_rows(g, act, "gate")
        if u.shape != g.shape or wt.numel() != act.in_features:
            raise ValueError("gate, up and norm weight shapes do not match")
        self._bind_stream()
        _hip.check(self.lib.rt_act_relu2_mul_norm_quantize(self.ctx, g.data_ptr(), u.data_ptr(), wt.data_ptr(),
                                                           float(eps), g.shape[0], act.handle,
                                                           a_out.data_ptr() if a_out is not None else None),
                   "rt_act_relu2_mul_norm_quantize")
        act.tokens = g.shape[0]
        return act

    def linear_act(self, w: DeviceTernaryWeights, act: DeviceActivations, out=None, residual=None):
        """y [M, N] fp32 = W2A8 linear of the activations held (+ residual [M, N])."""
        torch = _torch()
        if act.in_features != w.in_features:
            raise ValueError("activations and weights disagree on in_features")
        y = out if out is not None else torch.empty((act.tokens, w.out_features), dtype=torch.float32,
                                                    device=self.device)
        self._bind_stream()
        res = residual.data_ptr() if residual is not None else None
        _hip.check(self.lib.rt_linear_act_f32(self.ctx, w.handle, act.handle, res, y.data_ptr()), "rt_linear_act_f32")
        return y

    def plan_act(self, weights, acts, M: int, ys) -> LinearPlan:
        """One launch of len(weights) linears over caller-filled activations."""
        G = len(weights)
        if not (G == len(acts) == len(ys)) or G == 0:
            raise ValueError("plan_act needs equal, non-zero numbers of weights, activations and outputs")
        for w, a, y in zip(weights, acts, ys):
            if a.in_features != w.in_features or tuple(y.shape) != (M, w.out_features) or not y.is_contiguous():
                raise ValueError("plan_act: shapes do not match")
        P = ctypes.c_void_p
        wa = (P * G)(*[w.handle for w in weights])
        aa = (P * G)(*[a.handle for a in acts])
        ya = (P * G)(*[y.data_ptr() for y in ys])
        h = ctypes.c_void_p()
        _hip.check(self.lib.rt_plan_create_act(self.ctx, G, wa, aa, int(M), ya, ctypes.byref(h)), "rt_plan_create_act")
        return LinearPlan(self, h, (list(weights), list(acts), list(ys)))

    def plan_act_gate_up(self, w_gu, scales, act, M: int, a) -> LinearPlan:
        """Gate and up for M > 64 tokens over caller-filled activations in one GEMM launch
        (rt_plan_create_act_gate_up) on the matrix of interleave_gate_up: a fp32 [M, F] =
        relu(g)^2 * u, the values act_relu2_mul_quantize forms from separate g and u."""
        torch = _torch()
        N, K = w_gu.out_features, w_gu.in_features
        if act.in_features != K or a.dtype != torch.float32 or tuple(a.shape) != (M, N // 2) or not a.is_contiguous():
            raise ValueError("plan_act_gate_up: shapes do not match")
        h = ctypes.c_void_p()
        s_gate, s_up = scales
        _hip.check(self.lib.rt_plan_create_act_gate_up(self.ctx, w_gu.handle, float(s_gate), float(s_up), act.handle,
                                                       int(M), a.data_ptr(), ctypes.byref(h)),
                   "rt_plan_create_act_gate_up")
        return LinearPlan(self, h, (w_gu, act, a))

    def plan_fused(self, weights, mode: int, x, aux=None, aux2=None, eps: float = 1e-6, ys=None, residuals=None,
                   attn_head_dim: int = 0, attn_max_len: int = 0):
        """One-token plan whose single launch quantises its input row in the prologue:
        mode = _hip.SRC_QUANT / SRC_RMSNORM / SRC_RELU2MUL / SRC_RELU2MUL_NORM; x, aux, aux2
        device fp32 [K]; ys[g] fp32 [N_g] outputs (+ residuals[g])."""
        G = len(weights)
        if G == 0 or len(ys) != G or (residuals is not None and len(residuals) != G):
            raise ValueError("plan_fused: mismatched argument lists")
        K = weights[0].in_features
        for w, y in zip(weights, ys):
            if w.in_features != K or y.numel() != w.out_features or not y.is_contiguous():
                raise ValueError("plan_fused: shapes do not match")
        self._check_src(mode, K, x, aux, aux2, "plan_fused")
        if mode == _hip.SRC_ATTN_NORM:
            need = self.lib.rt_attention_decode_workspace(K // max(attn_head_dim, 1), attn_head_dim, attn_max_len)
            if attn_head_dim <= 0 or x.numel() * x.element_size() < need:
                raise ValueError("plan_fused: attention partials buffer too small")
        src = _hip.RtSrc(int(mode), x.data_ptr(), aux.data_ptr() if aux is not None else None,
                         aux2.data_ptr() if aux2 is not None else None, float(eps), int(attn_head_dim),
                         int(attn_max_len))
        P = ctypes.c_void_p
        wa = (P * G)(*[w.handle for w in weights])
        ya = (P * G)(*[y.data_ptr() for y in ys])
        ra = (P * G)(*[r.data_ptr() if r is not None else None for r in residuals]) if residuals is not None else None
        h = ctypes.c_void_p()
        _hip.check(self.lib.rt_plan_create_fused(self.ctx, G, wa, ctypes.byref(src), ya, ra, ctypes.byref(h)),
                   "rt_plan_create_fused")
        return LinearPlan(self, h, (list(weights), [x, aux, aux2], list(ys), list(residuals or [])))

    def _check_src(self, mode, K, x, aux, aux2, who):
        for t in ((x if mode != _hip.SRC_ATTN_NORM else None), aux,
                  (aux2 if mode != _hip.SRC_RMSNORM_SSQ else None)):
            if t is not None and (t.numel() < K or not t.is_contiguous() or t.device != self.device):
                raise ValueError(f"{who}: source tensors must be contiguous device tensors of >= K elements")
        if mode == _hip.SRC_RMSNORM_SSQ:
            t = aux2
            if (t is None or t.dtype != _torch().float64 or t.numel() < K // 32 or not t.is_contiguous()
                    or t.device != self.device):
                raise ValueError(f"{who}: RMSNORM_SSQ needs aux2 = float64 device partial sums [K/32]")

    def interleave_gate_up(self, w_gate, w_up):
        """The matrix rt_plan_create_gate_up runs: gate and up [F, K] interleaved in groups
        of 32 rows (rows 64 j .. 64 j + 31 = gate rows 32 j .., the next 32 = up rows 32 j ..),
        uploaded once; returns (matrix, (gate scale, up scale))."""
        F, K = w_gate.out_features, w_gate.in_features
        if (w_up.out_features, w_up.in_features) != (F, K) or F % 32:
            raise ValueError("interleave_gate_up: gate and up must have the same shape with F % 32 == 0")
        g, u = w_gate.download(), w_up.download()
        gu = np.stack([g.reshape(F // 32, 32, -1), u.reshape(F // 32, 32, -1)], axis=1).reshape(2 * F, -1)
        return self.upload(gu, K, 1.0), (w_gate.scale, w_up.scale)

    def plan_gate_up(self, w_gu, scales, mode: int, x, aux=None, aux2=None, eps: float = 1e-6, a=None, ssq=None,
                     g_out=None, u_out=None):
        """One-token gate/up plan of the gated FFN (rt_plan_create_gate_up) on the matrix of
        interleave_gate_up: a[i] = relu(g_i)^2 * u_i (fp32 [F]) and ssq[j] (float64 [F/32]) =
        sum of a^2 over outputs 32 j .. 32 j + 31, the input of an SRC_RMSNORM_SSQ plan."""
        torch = _torch()
        N, K = w_gu.out_features, w_gu.in_features
        F = N // 2
        if N % 64:
            raise ValueError("plan_gate_up: the interleaved matrix needs N % 64 == 0")
        self._check_src(mode, K, x, aux, aux2, "plan_gate_up")
        if a is None or a.numel() < F or a.dtype != torch.float32 or not a.is_contiguous():
            raise ValueError("plan_gate_up: a must be a contiguous float32 device tensor of F elements")
        if ssq is None or ssq.numel() < F // 32 or ssq.dtype != torch.float64 or not ssq.is_contiguous():
            raise ValueError("plan_gate_up: ssq must be a contiguous float64 device tensor of F/32 elements")
        for t in (g_out, u_out):
            if t is not None and (t.numel() < F or t.dtype != torch.float32 or not t.is_contiguous()):
                raise ValueError("plan_gate_up: g_out / u_out must be float32 device tensors of F elements")
        ptr = lambda t: t.data_ptr() if t is not None else None
        src = _hip.RtSrc(int(mode), x.data_ptr(), ptr(aux), ptr(aux2), float(eps), 0, 0)
        h = ctypes.c_void_p()
        s_gate, s_up = scales
        _hip.check(self.lib.rt_plan_create_gate_up(self.ctx, w_gu.handle, float(s_gate), float(s_up), ctypes.byref(src),
                                                   a.data_ptr(), ssq.data_ptr(), ptr(g_out), ptr(u_out),
                                                   ctypes.byref(h)), "rt_plan_create_gate_up")
        return LinearPlan(self, h, ([w_gu], [x, aux, aux2], [a, ssq], [g_out, u_out]))

    # -- KV cache in 4 bits (rt_kv4_*) ---------------------------------------------
    def kv4_cache(self, n_kv_heads: int, head_dim: int, max_len: int, batch: int = 1):
        """One layer's 4-bit KV cache for `batch` sequences of up to max_len positions: a uint8
        device tensor [batch, n_kv_heads, ceil(max_len / 64), 72 * head_dim] (its bytes are
        opaque).  Positions that nothing was written to read as NaN: a row that attends past what
        was appended is NaN, not a number from old memory."""
        if not self.lib.rt_kv4_bytes(int(batch), int(n_kv_heads), int(head_dim), int(max_len)):
            raise ValueError("kv4_cache: needs head_dim 64 or 128, batch * n_kv_heads <= 2^24, 1 <= max_len <= 2^20")
        torch = _torch()
        return torch.full((int(batch), int(n_kv_heads), (int(max_len) + 63) // 64, 18 * int(head_dim)), 0x7FC00000,
                          dtype=torch.int32, device=self.device).view(torch.uint8)  # (a scale's z = NaN, h = 0)

    # A step of decoding is a few microseconds of GPU work, so these calls look at each tensor once, touch
    # nothing that is already as the library takes it, and compare devices by their numbers.
    def _kv4_check(self, who, torch, cache, pos, max_len):
        """(B, Hkv, hd, Lmax) of a cache and its positions."""
        shape = cache.shape
        if (cache.dtype is not torch.uint8 or len(shape) != 4 or not cache.is_contiguous()
                or cache.get_device() != self.device_index or shape[3] not in (72 * 64, 72 * 128)):
            raise ValueError(f"{who}: cache must be a contiguous uint8 [B, Hkv, blocks, 72 * head_dim] tensor on the "
                             "backend's device (kv4_cache)")
        B, Hkv, blocks, size = shape
        Lmax = 64 * blocks if max_len is None else int(max_len)
        if not 64 * (blocks - 1) < Lmax <= 64 * blocks:
            raise ValueError(f"{who}: max_len {Lmax} does not fit a cache of {blocks} blocks of 64 positions")
        if (pos.dtype is not torch.int32 or pos.shape != (B,) or pos.get_device() != self.device_index
                or not pos.is_contiguous()):
            raise ValueError(f"{who}: pos must be a contiguous int32 [{B}] tensor on the backend's device")
        return B, Hkv, size // 72, Lmax

    def _kv4_rows(self, who, q, B, Hkv, hd):
        """(M, H) of q [B, M, H, hd]."""
        shape = q.shape
        if len(shape) != 4 or shape[0] != B or shape[3] != hd or shape[2] % max(Hkv, 1) or 0 in shape:
            raise ValueError(f"{who}: q of shape {tuple(shape)} does not fit a cache of {B} sequences, {Hkv} KV heads of {hd}")
        return shape[1], shape[2]

    def _kv4_new(self, who, q, k, v, rope, B, Hkv, hd, Lmax, max_len):
        """(Lmax, M, H) of new rows and their angles."""
        table = rope.shape
        if max_len is None and len(table) == 3:
            Lmax = min(Lmax, max(table[0], Lmax - 63))
        M, H = self._kv4_rows(who, q, B, Hkv, hd)
        if k.shape != (B, M, Hkv, hd) or v.shape != (B, M, Hkv, hd):
            raise ValueError(f"{who}: k and v must be {[B, M, Hkv, hd]}")
        if len(table) != 3 or table[1:] != (hd // 2, 2) or table[0] < Lmax:
            raise ValueError(f"{who}: rope must be [>= {Lmax}, {hd // 2}, 2]")
        return Lmax, M, H

    def _kv4_workspace(self, torch, B, M, H, Hkv, hd, Lmax):
        need = _kv4_workspace_bytes(B, M, H, Hkv, hd, Lmax)
        return need, torch.empty(need, dtype=torch.uint8, device=self.device) if need else None

    def _kv4_run(self, torch, name, fn, *args):
        """fn(ctx, *args) on the current stream (taken as the number it is: making a Stream object of it
        costs as much as a small launch)."""
        rc = self.lib.rt_ctx_set_stream(self.ctx, torch._C._cuda_getCurrentRawStream(self.device_index))
        rc = rc or fn(self.ctx, *args)
        if rc:
            _hip.check(rc, name)

    def _kv4_in(self, torch, x):
        """float32 device tensor, contiguous and 16-byte aligned (a copy where x is not)."""
        if not (isinstance(x, torch.Tensor) and x.dtype is torch.float32 and x.get_device() == self.device_index
                and x.is_contiguous()):
            x = self._dev(x, torch.float32)
        return x.clone() if x.data_ptr() & 15 else x

    def _kv4_out(self, who, torch, out, like, *others):
        """out, or a new tensor of like's shape; out may be like, and lies in none of the others."""
        if out is None:
            return torch.empty_like(like)
        if (out.dtype is not torch.float32 or out.shape != like.shape or not out.is_contiguous()
                or out.get_device() != self.device_index):
            raise ValueError(f"{who}: the output must be a contiguous float32 {list(like.shape)} tensor on the backend's "
                             "device")
        at, end = out.data_ptr(), out.data_ptr() + 4 * out.numel()
        for x in (like, *others):
            if x.data_ptr() < end and at < x.data_ptr() + x.numel() * x.element_size() and not (x is like and x.data_ptr() == at):
                raise ValueError(f"{who}: the output must not share memory with the other arguments (but may be q)")
        return out

    def kv4_append(self, q, k, v, cache, rope, pos, max_len=None, q_out=None):
        """RoPE of q [B, M, H, hd] and k [B, M, Hkv, hd], then k and v into the 4-bit cache at
        positions pos[b] + m (rt_kv4_append); rope float32 [>= max_len, hd / 2, 2].  Returns the
        rotated q (q_out, which may be q).  max_len: the cache's positions, where they are fewer
        than its blocks hold (None: as many as the blocks and rope hold; kv4_read and
        kv4_attention do not see rope, and take what the blocks hold: pass max_len to all of them
        where it is no multiple of 64).  Rows outside [0, max_len) are not written; their q is 0.
        For inference: gradients do not pass."""
        torch = _torch()
        B, Hkv, hd, Lmax = self._kv4_check("kv4_append", torch, cache, pos, max_len)
        q, k, v, rope = (self._kv4_in(torch, x) for x in (q, k, v, rope))
        Lmax, M, H = self._kv4_new("kv4_append", q, k, v, rope, B, Hkv, hd, Lmax, max_len)
        out = self._kv4_out("kv4_append", torch, q_out, q, k, v, rope, cache, pos)
        self._kv4_run(torch, "rt_kv4_append", self.lib.rt_kv4_append, q.data_ptr(), k.data_ptr(), v.data_ptr(), rope.data_ptr(),
                      cache.data_ptr(), out.data_ptr(), B, M, H, Hkv, hd, Lmax, pos.data_ptr())
        return out

    def kv4_step(self, q, k, v, cache, rope, pos, max_len=None, out=None):
        """A decoding step (q [B, 1, H, hd], k and v [B, 1, Hkv, hd], H / Hkv <= 16): kv4_append and
        kv4_attention of its q in one launch (rt_kv4_step), with the same results; out may be q."""
        torch = _torch()
        B, Hkv, hd, Lmax = self._kv4_check("kv4_step", torch, cache, pos, max_len)
        q, k, v, rope = (self._kv4_in(torch, x) for x in (q, k, v, rope))
        Lmax, M, H = self._kv4_new("kv4_step", q, k, v, rope, B, Hkv, hd, Lmax, max_len)
        if M != 1 or H > 16 * Hkv:
            raise ValueError("kv4_step: takes one token a sequence, and H / Hkv <= 16")
        out = self._kv4_out("kv4_step", torch, out, q, k, v, rope, cache, pos)
        need, ws = self._kv4_workspace(torch, B, 1, H, Hkv, hd, Lmax)
        self._kv4_run(torch, "rt_kv4_step", self.lib.rt_kv4_step, q.data_ptr(), k.data_ptr(), v.data_ptr(), rope.data_ptr(),
                      cache.data_ptr(), out.data_ptr(), B, H, Hkv, hd, Lmax, pos.data_ptr(),
                      ws.data_ptr() if need else None, need)
        return out

    def kv4_read(self, cache, pos, length: int, max_len=None):
        """The values that a 4-bit cache holds at positions pos[b] + (0 .. length - 1): (k, v)
        float32 [B, Hkv, length, hd]; zeros outside [0, max_len) (rt_kv4_read)."""
        torch = _torch()
        B, Hkv, hd, Lmax = self._kv4_check("kv4_read", torch, cache, pos, max_len)
        length = operator.index(length)
        if not 0 < length <= Lmax:
            raise ValueError(f"kv4_read: length {length} of a cache of {Lmax} positions")
        k = torch.empty((B, Hkv, length, hd), dtype=torch.float32, device=self.device)
        v = torch.empty_like(k)
        self._kv4_run(torch, "rt_kv4_read", self.lib.rt_kv4_read, cache.data_ptr(), k.data_ptr(), v.data_ptr(), B, length, Hkv, hd,
                      Lmax, pos.data_ptr())
        return k, v

    def kv4_attention(self, q, cache, pos, max_len=None, out=None):
        """Causal GQA attention of q [B, M, H, hd] (rotated, as kv4_append returns it) at positions
        pos[b] + m over a 4-bit cache (rt_kv4_attention): float32 [B, M, H, hd] (out, which may be
        q).  Rows outside [0, max_len) are 0.  For inference: gradients do not pass."""
        torch = _torch()
        B, Hkv, hd, Lmax = self._kv4_check("kv4_attention", torch, cache, pos, max_len)
        q = self._kv4_in(torch, q)
        M, H = self._kv4_rows("kv4_attention", q, B, Hkv, hd)
        out = self._kv4_out("kv4_attention", torch, out, q, cache, pos)
        need, ws = self._kv4_workspace(torch, B, M, H, Hkv, hd, Lmax)
        self._kv4_run(torch, "rt_kv4_attention", self.lib.rt_kv4_attention, q.data_ptr(), cache.data_ptr(), out.data_ptr(), B, M, H,
                      Hkv, hd, Lmax, pos.data_ptr(), ws.data_ptr() if need else None, need)
        return out

    # -- KV cache in pages (rt_paged_*) --------------------------------------------
    def paged_cache(self, n_kv_heads: int, head_dim: int, n_pages: int, page: int = 64, dtype=None):
        """One layer's paged KV cache: a tensor [2 (keys, values), n_pages, n_kv_heads, page, head_dim] of
        torch.bfloat16 (default), float16 or float32.  Which sequence has which pages is the caller's: calls take a
        table int32 [B, P] of page numbers and lens int32 [B], the slots that each sequence holds.  Slots
        that nothing was written to read as NaN.  Any tensor of this form does (a layer of a
        larger one too: the two outer dimensions may have any strides)."""
        torch = _torch()
        dtype = torch.bfloat16 if dtype is None else dtype
        if dtype not in _paged_types() or head_dim not in (64, 128) or page not in (16, 32, 64, 128, 256) or n_kv_heads < 1 or n_pages < 1:
            raise ValueError("paged_cache: needs head_dim 64 or 128, page 16, 32, 64, 128 or 256, bfloat16, float16 or float32")
        return torch.full((2, int(n_pages), int(n_kv_heads), page, head_dim), float("nan"), dtype=dtype, device=self.device)

    # (As with the calls above: each tensor is looked at once, and what is as the library takes it is not touched.)
    def _paged_int(self, who, torch, name, x, B):
        if (x.dtype is not torch.int32 or x.get_device() != self.device_index or not x.is_contiguous() or x.shape != (B,)):
            raise ValueError(f"{who}: {name} must be a contiguous int32 [{B}] tensor on the backend's device")
        return x.data_ptr()

    def _paged_table(self, who, torch, name, x):
        """[B, P] of a table."""
        shape = x.shape
        if x.dtype is not torch.int32 or x.get_device() != self.device_index or not x.is_contiguous() or len(shape) != 2:
            raise ValueError(f"{who}: {name} must be a contiguous int32 [B, P] tensor on the backend's device")
        return shape

    def _paged_check(self, who, torch, cache, table, lens):
        """(rt_pages, (type, Hkv, page, hd, B, P), bytes that the cache's pages span) of a cache, its table and lengths."""
        shape, strides, kind = cache.shape, cache.stride(), _paged_types().get(cache.dtype)
        if kind is None or len(shape) != 5 or shape[0] != 2 or cache.get_device() != self.device_index:
            raise ValueError(f"{who}: cache must be a bfloat16, float16 or float32 [2, pages, Hkv, page, head_dim] tensor on the "
                             "backend's device (paged_cache)")
        _, pages, Hkv, page, hd = shape
        rows = Hkv * page * hd
        if strides[4] != 1 or strides[3] != hd or (strides[2] != page * hd and Hkv > 1):
            raise ValueError(f"{who}: a page's [Hkv, page, head_dim] must be contiguous")
        B, P = self._paged_table(who, torch, "table", table)
        apart, step = strides[0], strides[1] if pages > 1 else rows
        return (_hip.PAGES.pack(cache.data_ptr(), apart, step, table.data_ptr(), self._paged_int(who, torch, "lens", lens, B), kind, pages,
                                Hkv, page, hd, B, P),
                (kind, Hkv, page, hd, B, P), (apart + (pages - 1) * step + rows) * (2 if kind else 4))

    def _paged_in(self, torch, x):
        """x as the library takes it: itself, or as _kv4_in copies it."""
        if isinstance(x, torch.Tensor) and x.dtype is torch.float32 and x.get_device() == self.device_index and x.is_contiguous():
            at = x.data_ptr()
            if not at & 15:
                return x, at
        x = self._kv4_in(torch, x)
        return x, x.data_ptr()

    def _paged_new(self, who, torch, q, k, v, rope, pos, counts, interleaved, sizes):
        """(rt_paged_new, q, (M, H), the other tensors that it names) of new tokens."""
        _, Hkv, _, hd, B, _ = sizes
        (q, at_q), (k, at_k), (v, at_v), (rope, at_rope) = (self._paged_in(torch, q), self._paged_in(torch, k),
                                                            self._paged_in(torch, v), self._paged_in(torch, rope))
        M, H = self._kv4_rows(who, q, B, Hkv, hd)
        rows = (B, M, Hkv, hd)
        if k.shape != rows or v.shape != rows:
            raise ValueError(f"{who}: k and v must be {list(rows)}")
        table = rope.shape
        if len(table) != 3 or table[2] != 2 or table[1] % 4 or not 0 < 2 * table[1] <= hd or not table[0]:
            raise ValueError(f"{who}: rope must be [positions, rotary / 2, 2], rotary a multiple of 8 up to head_dim")
        new = _hip.PAGED_NEW.pack(at_q, at_k, at_v, at_rope, self._paged_int(who, torch, "pos", pos, B),
                                  self._paged_int(who, torch, "counts", counts, B) if counts is not None else 0, table[0], 2 * table[1],
                                  bool(interleaved), M, H)
        return new, q, (M, H), (k, v, rope, pos) if counts is None else (k, v, rope, pos, counts)

    def _paged_apart(self, who, name, x, cache, span, *others):
        """x, which the call writes, lies in none of the others."""
        at = x.data_ptr()
        end = at + x.numel() * x.element_size()
        first = cache.data_ptr()
        if first < end and at < first + span:
            raise ValueError(f"{who}: {name} must not share memory with the cache")
        for y in others:
            first = y.data_ptr()
            if first < end and at < first + y.numel() * y.element_size():
                raise ValueError(f"{who}: {name} must not share memory with the other arguments")

    def _paged_weights(self, who, torch, weights, sizes):
        """The slots of a row of accumulated weights."""
        _, Hkv, page, _, B, P = sizes
        shape = weights.shape
        if (weights.dtype is not torch.float32 or len(shape) != 3 or shape[0] != B or shape[1] != Hkv or shape[2] < P * page
                or not weights.is_contiguous() or weights.get_device() != self.device_index):
            raise ValueError(f"{who}: weights must be a contiguous float32 [{B}, {Hkv}, >= {P * page}] tensor on the backend's device")
        return shape[2]

    def paged_append(self, q, k, v, cache, table, lens, rope, pos, counts=None, interleaved: bool = False, q_out=None):
        """RoPE of q [B, M, H, hd] and k [B, M, Hkv, hd], then k and v into the paged cache at slots lens[b] + m
        (rt_paged_append).  Token m stands at position pos[b] + m (which runs ahead of the slots once a
        cache was cut); rope float32 [positions, rotary / 2, 2] (rope_table) turns a head's first `rotary` dimensions: pairs (i,
        i + rotary / 2), or (2 i, 2 i + 1) with interleaved.  counts int32 [B]: a sequence's tokens where they are
        fewer than M.  Returns the rotated q (q_out, which may be q).  Tokens past counts, without a row of rope or without a
        slot are not written; their q is 0.  lens is not changed.  For inference: gradients do not pass."""
        torch = _torch()
        pages, sizes, span = self._paged_check("paged_append", torch, cache, table, lens)
        new, q, _, others = self._paged_new("paged_append", torch, q, k, v, rope, pos, counts, interleaved, sizes)
        if q_out is None:
            out = torch.empty_like(q)
        else:
            out = self._kv4_out("paged_append", torch, q_out, q, *others, table, lens)
            self._paged_apart("paged_append", "q_out", out, cache, span)
        self._kv4_run(torch, "rt_paged_append", self.lib.rt_paged_append, pages, new, out.data_ptr())
        return out

    def paged_attention(self, q, cache, table, lens, weights=None, out=None):
        """Attention of one token a sequence, q [B, 1, H, hd] (rotated, as paged_append returns it), over the lens[b] slots
        of a paged cache (rt_paged_attention): float32 [B, 1, H, hd] (out, which may be q); zeros for a sequence
        without slots.  weights float32 [B, Hkv, slots]: what every slot weighed (the softmax's weights, summed over a KV head's
        query heads) is added to it, for paged_evict.  (With weights the output may differ in its last bits: another order of
        additions; and memory of 4 bytes for every head and slot of the table, so give a table no wider than the longest sequence
        needs.  Up to 1024 sequences are cut into pieces that run side by side; in a larger batch the longest decides.)  For
        inference: gradients do not pass."""
        torch = _torch()
        pages, sizes, span = self._paged_check("paged_attention", torch, cache, table, lens)
        q, at = self._paged_in(torch, q)
        M, H = self._kv4_rows("paged_attention", q, sizes[4], sizes[1], sizes[3])
        if M != 1:
            raise ValueError("paged_attention: takes one token a sequence")
        out, args = self._paged_attend("paged_attention", torch, out, q, cache, span, sizes, H, weights, (table, lens))
        self._kv4_run(torch, "rt_paged_attention", self.lib.rt_paged_attention, pages, at, H, *args[1:])
        return out

    def paged_step(self, q, k, v, cache, table, lens, rope, pos, interleaved: bool = False, weights=None, out=None):
        """A decoding step (q [B, 1, H, hd], k and v [B, 1, Hkv, hd]): paged_append, then paged_attention of its q over the
        lens[b] + 1 slots there are then, in one call (rt_paged_step).  A token without a row of rope or without a slot
        attends to nothing.  lens is not changed: the next step's is lens + 1."""
        torch = _torch()
        pages, sizes, span = self._paged_check("paged_step", torch, cache, table, lens)
        new, q, (M, H), others = self._paged_new("paged_step", torch, q, k, v, rope, pos, None, interleaved, sizes)
        if M != 1:
            raise ValueError("paged_step: takes one token a sequence")
        out, args = self._paged_attend("paged_step", torch, out, q, cache, span, sizes, H, weights, (*others, table, lens))
        self._kv4_run(torch, "rt_paged_step", self.lib.rt_paged_step, pages, new, *args[1:])
        return out

    def _paged_attend(self, who, torch, out, q, cache, span, sizes, H, weights, others):
        """(out, (workspace, the arguments that follow the queries))."""
        if out is None:
            out = torch.empty_like(q)
        else:
            out = self._kv4_out(who, torch, out, q, *others)
            self._paged_apart(who, "out", out, cache, span)
        at, slots = None, 0
        if weights is not None:
            slots, at = self._paged_weights(who, torch, weights, sizes), weights.data_ptr()
            self._paged_apart(who, "weights", weights, cache, span, q, out, *others)
        need = _paged_workspace_bytes(*sizes, H, slots > 0)
        if not need:
            return out, (None, at, slots, out.data_ptr(), None, 0)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        return out, (ws, at, slots, out.data_ptr(), ws.data_ptr(), need)

    def paged_evict(self, cache, table, lens, weights, keep: int, recent: int, new_table):
        """Cuts every sequence of a paged cache to `keep` slots (rt_paged_evict): for each KV head the last `recent` and, of
        those before them, the ones with the largest weights (ties: the lowest slot), in their order.  Their keys and values
        are copied to the pages of new_table int32 [B, new_P], which must be pages that no table of these sequences holds;
        the old ones stay as they were and are free afterwards.  Returns (kept int32 [B, Hkv, keep]: the slots, -1 behind the
        last; new_lens int32 [B]; new_weights, shaped as weights: the kept slots', then zeros; to go on with them over a new_table of
        more slots, give weights with rows for new_P * page).  Sequences of no more than `keep` slots move as they are."""
        torch = _torch()
        pages, sizes, span = self._paged_check("paged_evict", torch, cache, table, lens)
        _, Hkv, page, _, B, _ = sizes
        slots = self._paged_weights("paged_evict", torch, weights, sizes)
        keep, recent = operator.index(keep), operator.index(recent)
        new_B, new_P = self._paged_table("paged_evict", torch, "new_table", new_table)
        if new_B != B:
            raise ValueError(f"paged_evict: new_table must be int32 [{B}, new_P]")
        if not (0 <= recent <= keep and 0 < keep <= new_P * page):
            raise ValueError(f"paged_evict: keep {keep} and recent {recent}: needs 0 <= recent <= keep, and pages for keep >= 1 slots")
        self._paged_apart("paged_evict", "new_table", new_table, cache, span, table)
        self._paged_apart("paged_evict", "weights", weights, cache, span)
        kept = torch.empty((B, Hkv, keep), dtype=torch.int32, device=self.device)
        new_lens, new_weights = torch.empty_like(lens), torch.empty_like(weights)
        need = _paged_evict_workspace_bytes(*sizes)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        self._kv4_run(torch, "rt_paged_evict", self.lib.rt_paged_evict, pages, weights.data_ptr(), slots, keep, recent,
                      new_table.data_ptr(), new_P, kept.data_ptr(), new_lens.data_ptr(), new_weights.data_ptr(),
                      ws.data_ptr() if need else None, need)
        return kept, new_lens, new_weights

    def __del__(self):
        try:
            if getattr(self, "ctx", None):
                self.lib.rt_ctx_destroy(self.ctx)
                self.ctx = None
        except Exception:
            pass


__all__ = ["HIPTernaryOps", "DeviceTernaryWeights", "DeviceActivations", "LinearPlan", "unpack_rotor_rows"]
