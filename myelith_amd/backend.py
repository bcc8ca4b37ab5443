"""RocmBackend: the host-side mirror of the reference's `Backend` trait.

Mirrors INTEGER_LLM/kernels/src/backends/rocm.rs (RocmBackend::init, name,
hardware_family, feature_tag, gcn_arch) and the trait methods of
INTEGER_LLM/kernels/src/backend.rs:23-127, plus the free functions that
runtime/src/model.rs calls directly (linear_w8a16_pc, add_bias_i16,
argmax_int).  Every method calls libmyl_hip.so; arguments keep the reference's
names, order and meaning.  Shape errors raise ValueError where the reference
panics.

The `*_dev` methods take torch tensors already on the GPU and run on torch's
current stream (plumbing only: the arithmetic is in the HIP kernels).
"""
from __future__ import annotations

import ctypes as C
import weakref

import numpy as np

from ._lib import MYL_E_INVALID, lib


class MylError(RuntimeError):
    pass


def _a(x, dtype) -> np.ndarray:
    return np.ascontiguousarray(np.asarray(x), dtype=dtype)


def _p(a):
    return None if a is None else a.ctypes.data


def _need(ok, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _need_dev(what: str, device, **tensors) -> None:
    """name=(tensor, dtype name, shape): on the device, of that type and shape, its
    elements in order (strides are the caller's to check where shape is None)."""
    import torch
    for name, (t, dtype, shape) in tensors.items():
        if t.device != device or t.dtype is not getattr(torch, dtype):
            raise ValueError(f"{what}: {name} must be {dtype} on {device}")
        if shape is not None and not (t.shape == shape and t.is_contiguous()):
            raise ValueError(f"{what}: {name} must be contiguous {list(shape)}, not {list(t.shape)}")


def _need_bytes(what: str, **values) -> None:
    """Numbers that the library takes as uint8, which would keep the low bits of others."""
    for name, v in values.items():
        if not 0 <= v <= 255:
            raise ValueError(f"{what}: {name} must be 0 to 255, not {v}")


def _strides(t):
    """The strides that an element's place depends on (None for dimensions of one element or
    none, whose stride says nothing)."""
    st, shape = t.stride(), t.shape
    if 0 in shape:
        return (None,) * len(st)
    return tuple(s if n > 1 else None for s, n in zip(st, shape)) if 1 in shape else st


def _apart(what: str, name: str, stride, dense: int) -> int:
    """The stride of a dimension, `dense` where it says nothing.  0 is refused: an expanded
    tensor owns fewer elements than a kernel would take it for."""
    if stride is None:
        return dense
    if stride == 0:
        raise ValueError(f"{what}: {name} must not be expanded (a stride of 0)")
    return stride


class RocmBackend:
    """One HIP context on one device (rocm.rs:41-60)."""

    _own_stream = None  # the context's, until a caller's takes its place

    def __init__(self, device_id: int = 0):
        h = C.c_void_p()
        rc = lib().myl_init(device_id, C.byref(h))
        if rc != 0:
            raise MylError(f"RocmBackend::init({device_id}) failed with status {rc}")
        self._h = h
        self._device_id = device_id
        self._own_stream = lib().myl_stream(h)
        # models and MoE layers on this context: closed before it is destroyed,
        # whatever order the interpreter finalises them in
        self._owned = weakref.WeakSet()
        arch = C.create_string_buffer(128)
        cus = C.c_int()
        hbm = C.c_uint64()
        lib().myl_device_info(self._h, arch, 128, C.byref(cus), C.byref(hbm))
        self._arch = arch.value.decode()
        self.cu_count = cus.value
        self.hbm_bytes = hbm.value

    # ---- identity (rocm.rs:62-82) -------------------------------------------
    def device_id(self) -> int:
        return self._device_id

    def gcn_arch(self) -> str:
        return self._arch

    @staticmethod
    def name() -> str:
        return lib().myl_backend_name().decode()

    @staticmethod
    def hardware_family() -> str:
        return lib().myl_hardware_family().decode()

    @staticmethod
    def feature_tag() -> str:
        return lib().myl_feature_tag().decode()

    # ---- plumbing -------------------------------------------------------------
    @property
    def handle(self):
        return self._h

    def adopt(self, obj) -> None:
        """Registers an object holding device state of this context; close()
        closes it first."""
        self._owned.add(obj)

    def close(self) -> None:
        if self._h:
            for obj in list(self._owned):
                obj.close()
            lib().myl_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def check(self, rc: int, what: str) -> None:
        if rc != 0:
            msg = lib().myl_last_error(self._h).decode()
            if rc == MYL_E_INVALID:
                raise ValueError(f"{what}: {msg}")
            raise MylError(f"{what} failed ({rc}): {msg}")

    def synchronize(self) -> None:
        self.check(lib().myl_synchronize(self._h), "synchronize")

    def read_probe_dev(self, buf, out) -> None:
        """One pass of 16-byte nontemporal loads over the device tensor buf (a
        measurement of the achievable read rate; out: a device int32 word)."""
        self.check(lib().myl_read_probe(self._h, buf.data_ptr(), buf.numel() * buf.element_size(), out.data_ptr()),
                   "read_probe")

    def use_torch_stream(self) -> None:
        """Launch on torch's current HIP stream (so torch events time our kernels)."""
        import torch
        self.check(lib().myl_set_stream(self._h, C.c_void_p(torch.cuda.current_stream().cuda_stream)), "set_stream")

    # ---- Backend trait (backend.rs:39-126), host slices ----------------------------
    def linear_w8a16(self, x, W, in_features: int, out_features: int, w_shifts, act_frac: int, out_frac: int):
        x, W, ws = _a(x, np.int16), _a(W, np.int8), _a(w_shifts, np.uint8)
        if W.size != in_features * out_features or ws.size != out_features or x.size < in_features:
            raise ValueError("linear_w8a16: W does not hold out_features rows of in_features (linear.rs:51-58)")
        out = np.zeros(out_features, np.int16)
        self.check(lib().myl_linear_w8a16(self._h, _p(x), _p(W), _p(out), in_features, out_features, _p(ws),
                                          act_frac, out_frac), "linear_w8a16")
        return out

    def linear_w8a16_pc(self, x, W, in_features: int, w_shifts, act_frac: int, out_frac):
        x, W, ws, of = _a(x, np.int16), _a(W, np.int8), _a(w_shifts, np.uint8), _a(out_frac, np.uint8)
        n = ws.size
        if W.size != in_features * n or of.size != n or x.size < in_features:
            raise ValueError("linear_w8a16_pc: shape mismatch (linear.rs:95-107)")
        out = np.zeros(n, np.int16)
        self.check(lib().myl_linear_w8a16_pc(self._h, _p(x), _p(W), _p(out), in_features, n, _p(ws), act_frac,
                                             _p(of)), "linear_w8a16_pc")
        return out

    def add_bias_i16(self, out, bias, bias_shifts, out_frac: int):
        o, b, bs = _a(out, np.int16).copy(), _a(bias, np.int16), _a(bias_shifts, np.uint8)
        if o.size != b.size or b.size != bs.size:
            raise ValueError("add_bias_i16: out, bias and shifts must have the same length (linear.rs:133-140)")
        self.check(lib().myl_add_bias_i16(self._h, _p(o), _p(b), _p(bs), o.size, out_frac), "add_bias_i16")
        return o

    def rmsnorm(self, x, x_shifts, gamma, gamma_shifts, rsqrt_lut, lut_input_shift: int, lut_output_frac: int,
                inv_n_q20: int, out_frac: int):
        x, xs, g, gs = _a(x, np.int16), _a(x_shifts, np.uint8), _a(gamma, np.int8), _a(gamma_shifts, np.uint8)
        lut = _a(rsqrt_lut, np.int16)
        n = x.size
        if not (g.size == n and gs.size == n and xs.size == n):
            raise ValueError("rmsnorm: x, gamma, gamma_shifts and x_shifts must match (rmsnorm.rs:73-75)")
        out = np.zeros(n, np.int16)
        self.check(lib().myl_rmsnorm(self._h, _p(x), _p(xs), _p(g), _p(gs), n, _p(lut), lut.size, lut_input_shift,
                                     lut_output_frac, inv_n_q20, _p(out), out_frac), "rmsnorm")
        return out

    def softmax(self, logits, exp_lut, lut_shift: int, frac_bits: int):
        z, lut = _a(logits, np.int32), _a(exp_lut, np.int16)
        out = np.zeros(z.size, np.int32)
        self.check(lib().myl_softmax(self._h, _p(z), _p(out), z.size, _p(lut), lut.size, lut_shift, frac_bits),
                   "softmax")
        return out

    def attention(self, q, k, v, mask, score_mult: int, score_shift: int, exp_lut, lut_shift: int,
                  prob_frac: int):
        q, k, v = _a(q, np.int16), _a(k, np.int16), _a(v, np.int16)
        if q.ndim != 2 or k.shape != v.shape or k.shape[1] != q.shape[1]:
            raise ValueError("attention: q [q_len x hd], k and v [kv_len x hd] (attention.rs:53-56)")
        ql, hd = q.shape
        kl = k.shape[0]
        mk = None if mask is None else _a(mask, np.uint8)
        if mk is not None and mk.shape != (ql, kl):
            raise ValueError("attention: mask must be [q_len x kv_len]")
        lut = _a(exp_lut, np.int16)
        out = np.zeros((ql, hd), np.int16)
        self.check(lib().myl_attention(self._h, _p(q), _p(k), _p(v), _p(out), ql, kl, hd, _p(mk), score_mult,
                                       score_shift, _p(lut), lut.size, lut_shift, prob_frac), "attention")
        return out

    def rope(self, q, k, cos_lut, sin_lut, positions, frac_bits: int):
        q, k = _a(q, np.int16).copy(), _a(k, np.int16).copy()
        c, s, p = _a(cos_lut, np.int16), _a(sin_lut, np.int16), _a(positions, np.uint64)
        n, hd = q.shape
        if k.shape != q.shape or p.size != n:
            raise ValueError("rope: q, k and positions must agree")
        self.check(lib().myl_rope(self._h, _p(q), _p(k), n, hd, _p(c), _p(s), c.size, _p(p), frac_bits), "rope")
        return q, k

    def mlp(self, x, W_gate, W_up, W_down, gate_w_shifts, up_w_shifts, down_w_shifts, silu_lut, in_frac: int,
            gate_out_frac: int, up_out_frac: int, down_in_frac: int, silu_in_frac: int, silu_lut_offset: int,
            silu_out_frac: int, out_frac):
        x = _a(x, np.int16)
        hidden = x.size
        Wg, Wu, Wd = _a(W_gate, np.int8), _a(W_up, np.int8), _a(W_down, np.int8)
        inter = Wg.size // hidden  # rocm.rs:183-186
        gs, us, ds = _a(gate_w_shifts, np.uint8), _a(up_w_shifts, np.uint8), _a(down_w_shifts, np.uint8)
        silu, of = _a(silu_lut, np.int16), _a(out_frac, np.uint8)
        if Wg.size != inter * hidden or Wu.size != Wg.size or Wd.size != Wg.size or gs.size != inter \
                or us.size != inter or ds.size != hidden or of.size != hidden:
            raise ValueError("mlp: weight and shift shapes do not agree (mlp.rs:28-74)")
        out = np.zeros(hidden, np.int16)
        self.check(lib().myl_mlp(self._h, _p(x), _p(Wg), _p(Wu), _p(Wd), _p(out), hidden, inter, _p(gs), _p(us),
                                 _p(ds), _p(silu), silu.size, in_frac, gate_out_frac, up_out_frac, down_in_frac,
                                 silu_in_frac, silu_lut_offset, silu_out_frac, _p(of)), "mlp")
        return out

    def argmax_int(self, values) -> int:
        v = _a(values, np.int32)
        out = C.c_int64()
        self.check(lib().myl_argmax_int(self._h, _p(v), v.size, C.byref(out)), "argmax_int")
        return out.value

    def sample_integer_cdf(self, logits, state: int):
        """sampling.rs:27-46 on the GPU: (token, new_state)."""
        v = _a(logits, np.int32)
        tok, ns = C.c_int64(), C.c_uint64()
        self.check(lib().myl_sample_integer_cdf(self._h, _p(v), v.size, int(state) & (2**64 - 1), C.byref(tok),
                                                C.byref(ns)), "sample_integer_cdf")
        return int(tok.value), int(ns.value)

    # ---- device forms (torch tensors on the GPU) ------------------------------
    def linear_w8a16_dev(self, x, W, w_shifts, act_frac: int, out_frac: int = 0, out_frac_pc=None, out=None):
        M, K = x.shape
        N = W.shape[0]
        if out is None:
            import torch
            out = torch.empty((M, N), dtype=torch.int16, device=x.device)
        # small products are bound by this call: nothing is imported or wrapped
        # that the launch does not need
        rc = lib().myl_linear_w8a16_dev(self._h, x.data_ptr(), M, x.stride(0), W.data_ptr(), N, K, w_shifts.data_ptr(),
                                        act_frac, out_frac, None if out_frac_pc is None else out_frac_pc.data_ptr(),
                                        out.data_ptr(), out.stride(0))
        if rc:
            self.check(rc, "linear_w8a16_dev")
        return out

    def linear_w8a16_dev_noalloc(self, x, W, w_shifts, act_frac: int, out_frac: int = 0, out_frac_pc=None, out=None):
        """linear_w8a16_dev without device allocation: `out` must be given
        (the library allocates nothing; include/myl_hip.h states the limit)."""
        M, K = x.shape
        N = W.shape[0]
        assert out is not None and tuple(out.shape) == (M, N), "out [M x N] is the caller's"
        self.check(lib().myl_linear_w8a16_dev_noalloc(self._h, x.data_ptr(), M, x.stride(0), W.data_ptr(), N, K,
                                                      w_shifts.data_ptr(), act_frac, out_frac,
                                                      None if out_frac_pc is None else out_frac_pc.data_ptr(),
                                                      out.data_ptr(), out.stride(0)), "linear_w8a16_dev_noalloc")
        return out

    def linear_w8a16_mult_dev(self, x, W, mult, shift, out=None):
        M, K = x.shape
        N = W.shape[0]
        if out is None:
            import torch
            out = torch.empty((M, N), dtype=torch.int16, device=x.device)
        rc = lib().myl_linear_w8a16_mult_dev(self._h, x.data_ptr(), M, x.stride(0), W.data_ptr(), N, K, mult.data_ptr(),
                                             shift.data_ptr(), out.data_ptr(), out.stride(0))
        if rc:
            self.check(rc, "linear_w8a16_mult_dev")
        return out

    def logits_dev(self, x, W, row_shifts, norm_frac: int, logit_frac: int, out=None):
        import torch
        M, K = x.shape
        N = W.shape[0]
        bits = 16 if W.dtype == torch.int16 else 8
        if out is None:
            out = torch.empty((M, N), dtype=torch.int32, device=x.device)
        self.check(lib().myl_logits_dev(self._h, x.data_ptr(), M, x.stride(0), W.data_ptr(), bits, N, K,
                                        row_shifts.data_ptr(), norm_frac, logit_frac, out.data_ptr(), out.stride(0)),
                   "logits_dev")
        return out

    def dot_i8_i16_dev(self, x, W, out=None):
        M, K = x.shape
        N = W.shape[0]
        if out is None:
            import torch
            out = torch.empty((M, N), dtype=torch.int64, device=x.device)
        rc = lib().myl_dot_i8_i16_dev(self._h, x.data_ptr(), M, x.stride(0), W.data_ptr(), N, K, out.data_ptr(),
                                      out.stride(0))
        if rc:
            self.check(rc, "dot_i8_i16_dev")
        return out

    def rmsnorm_dev(self, x, x_shifts, gamma, gamma_shifts, rsqrt_lut, lut_input_shift, lut_output_frac, inv_n_q20,
                    out_frac, out=None):
        import torch
        M, n = x.shape
        if out is None:
            out = torch.empty_like(x)
        self.check(lib().myl_rmsnorm_dev(self._h, x.data_ptr(), M, x.stride(0), x_shifts.data_ptr(), gamma.data_ptr(),
                                         gamma_shifts.data_ptr(), n, rsqrt_lut.data_ptr(), rsqrt_lut.numel(),
                                         lut_input_shift, lut_output_frac, inv_n_q20, out_frac, out.data_ptr(),
                                         out.stride(0)), "rmsnorm_dev")
        return out

    def softmax_dev(self, z, exp_lut, lut_shift, frac_bits, out=None):
        import torch
        M, n = z.shape
        if out is None:
            out = torch.empty_like(z)
        self.check(lib().myl_softmax_dev(self._h, z.data_ptr(), M, n, z.stride(0), exp_lut.data_ptr(), exp_lut.numel(),
                                         lut_shift, frac_bits, out.data_ptr(), out.stride(0)), "softmax_dev")
        return out

    def argmax_dev(self, v, out=None):
        M, n = v.shape
        if out is None:
            import torch
            out = torch.empty(M, dtype=torch.int64, device=v.device)
        rc = lib().myl_argmax_dev(self._h, v.data_ptr(), M, n, v.stride(0), out.data_ptr())
        if rc:
            self.check(rc, "argmax_dev")
        return out

    def sample_dev(self, z, states, tokens=None, new_states=None):
        """Rows of sample_integer_cdf (sampling.rs:27-46): z int32 [M x n],
        states uint64 [M] (torch int64 tensors hold the bits)."""
        import torch
        M, n = z.shape
        if tokens is None:
            tokens = torch.empty(M, dtype=torch.int64, device=z.device)
        if new_states is None:
            new_states = torch.empty(M, dtype=torch.int64, device=z.device)
        self.check(lib().myl_sample_dev(self._h, z.data_ptr(), M, n, z.stride(0), states.data_ptr(), tokens.data_ptr(),
                                        new_states.data_ptr()), "sample_dev")
        return tokens, new_states

    def logsoftmax_dev(self, z, exp_lut, targets, out=None):
        """Integer log-softmax at targets[m] per row, Q16 int64 (build-defined;
        the reference's perplexity probe uses f64, perplexity_probe.rs:55-67)."""
        import torch
        M, n = z.shape
        lut = exp_lut if isinstance(exp_lut, torch.Tensor) else torch.from_numpy(
            np.ascontiguousarray(exp_lut, dtype=np.int16)).to(z.device)
        t = targets if isinstance(targets, torch.Tensor) else torch.as_tensor(
            np.asarray(targets, dtype=np.int64), device=z.device)
        if out is None:
            out = torch.empty(M, dtype=torch.int64, device=z.device)
        self.check(lib().myl_logsoftmax_dev(self._h, z.data_ptr(), M, n, z.stride(0), lut.data_ptr(), lut.numel(),
                                            t.data_ptr(), out.data_ptr()), "logsoftmax_dev")
        return out

    # ---- a serving step: adapters, a shared prefix, drafted tokens ---------------
    def _workspace(self, device, workspace, stream, size_of, *sizes):
        """The caller's workspace (the call checks its size), or one for this call alone."""
        if workspace is not None:
            if workspace.device != device or not workspace.is_contiguous():
                raise ValueError("workspace: contiguous, on the operands' device")
            return workspace
        return self._empty(max(size_of(self._h, *sizes), 1), "uint8", device, stream)

    @staticmethod
    def _empty(shape, dtype: str, device, stream):
        """A tensor that a call writes: its memory is handed on only when `stream`
        (_other_stream) has passed the call."""
        import torch
        t = torch.empty(shape, dtype=getattr(torch, dtype), device=device)
        if stream is not None:
            t.record_stream(stream)
        return t

    def _other_stream(self, device):
        """The context's stream where nothing orders it with torch's current one: not if
        they are the same, nor for the null stream and the context's own, which HIP makes
        wait for each other."""
        import torch
        if device.type != "cuda" or device.index != self._device_id:  # the call will be refused
            return None
        stream, torchs = lib().myl_stream(self._h) or 0, torch.cuda.current_stream(device).cuda_stream
        if stream == torchs or (torchs == 0 and stream == self._own_stream):
            return None
        return torch.cuda.ExternalStream(stream, device=device)

    @staticmethod
    def _after_last_use(what: str, device, stream) -> None:
        """Behind a call's allocations, before its launch: the last use of their memory may
        still be queued on torch's current stream, so the context's stream waits for it."""
        import torch
        torchs, captured = torch.cuda.current_stream(device), []
        for s in (stream, torchs):
            with torch.cuda.stream(s):  # its device's, whatever the current device
                captured.append(torch.cuda.is_current_stream_capturing())
        if captured[0] != captured[1]:
            raise ValueError(f"{what}: while one of torch's stream and the context's is captured, outputs and workspace are the caller's")
        stream.wait_stream(torchs)

    def _need_here(self, what: str, device) -> None:
        if device.type != "cuda" or device.index != self._device_id:
            raise ValueError(f"{what}: the operands must be on device {self._device_id}")

    @staticmethod
    def _new_workspace(nbytes: int, device, what: str):
        import torch
        _need(nbytes > 0, f"{what}: these sizes are not supported")
        return torch.empty(nbytes, dtype=torch.uint8, device=device)

    def linear_w8a16_adapters_workspace(self, x, W, A):
        """A workspace for linear_w8a16_adapters_dev on operands of these shapes, and on smaller ones."""
        n = lib().myl_linear_w8a16_adapters_workspace(self._h, x.shape[0], W.shape[0], x.shape[1], A.shape[1],
                                                      A.shape[0])
        return self._new_workspace(n, x.device, "linear_w8a16_adapters_dev")

    def linear_w8a16_adapters_dev(self, x, W, w_shifts, act_frac: int, ids, A, a_shifts, mid_frac: int, B, b_shifts,
                                  out_frac: int = 0, out_frac_pc=None, out=None, workspace=None):
        """linear_w8a16_dev plus each row's low-rank adapter: x int16 [M x K],
        W int8 [N x K], ids int32 [M] (an id outside [0, n): none), A int8
        [n x rank x K] with a_shifts uint8 [n x rank], B int8 [n x N x rank]
        with b_shifts uint8 [n x N] (include/myl_hip.h states the arithmetic)."""
        what = "linear_w8a16_adapters_dev"
        if (act_frac | mid_frac | out_frac) >> 8:
            _need_bytes(what, act_frac=act_frac, mid_frac=mid_frac, out_frac=out_frac)
        M, K = x.shape
        N = W.shape[0]
        n, rank = A.shape[:2]
        _need_dev(what, x.device, x=(x, "int16", None), W=(W, "int8", (N, K)), w_shifts=(w_shifts, "uint8", (N,)),
                  ids=(ids, "int32", (M,)), A=(A, "int8", (n, rank, K)), a_shifts=(a_shifts, "uint8", (n, rank)),
                  B=(B, "int8", (n, N, rank)), b_shifts=(b_shifts, "uint8", (n, N)))
        ldx, step = _strides(x)
        ldx = _apart(what, "x", ldx, K)
        if step not in (None, 1):
            raise ValueError(f"{what}: the elements of a row of x follow one another")
        if out_frac_pc is not None:
            _need_dev(what, x.device, out_frac_pc=(out_frac_pc, "uint8", (N,)))
        stream = self._other_stream(x.device) if out is None or workspace is None else None
        if out is None:
            out = self._empty((M, N), "int16", x.device, stream)
        _need_dev(what, x.device, out=(out, "int16", None))
        ldo, step = _strides(out)
        ldo = _apart(what, "out", ldo, N)
        if out.shape != (M, N) or step not in (None, 1):
            raise ValueError(f"{what}: out must be [M x N]")
        self._need_here(what, x.device)
        ws = self._workspace(x.device, workspace, stream, lib().myl_linear_w8a16_adapters_workspace, M, N, K, rank, n)
        if stream is not None:
            self._after_last_use(what, x.device, stream)
        rc = lib().myl_linear_w8a16_adapters_dev(
            self._h, x.data_ptr(), M, ldx, W.data_ptr(), N, K, w_shifts.data_ptr(), act_frac, out_frac,
            None if out_frac_pc is None else out_frac_pc.data_ptr(), ids.data_ptr(), A.data_ptr(), a_shifts.data_ptr(),
            mid_frac, B.data_ptr(), b_shifts.data_ptr(), n, rank, out.data_ptr(), ldo,
            ws.data_ptr(), ws.numel() * ws.element_size())
        if rc:
            self.check(rc, what)
        return out

    def attention_prefix_workspace(self, q, k_prefix, k_tail, rows_per_seq: int = 1, max_tail=None):
        """A workspace for attention_prefix_dev on operands of these shapes, and on smaller ones."""
        n = lib().myl_attention_prefix_workspace(self._h, q.shape[0] // max(1, rows_per_seq), rows_per_seq, q.shape[1],
                                                 k_prefix.shape[0], q.shape[2], k_prefix.shape[1],
                                                 k_tail.shape[2] if max_tail is None else max_tail)
        return self._new_workspace(n, q.device, "attention_prefix_dev")

    def attention_prefix_dev(self, q, k_prefix, v_prefix, k_tail, v_tail, lens, score_mult: int, score_shift: int,
                             exp_lut, lut_shift: int, prob_frac: int, rows_per_seq: int = 1, slots=None, max_tail=None,
                             out=None, workspace=None):
        """Attention of a batch behind a shared prefix, int16 throughout: q and out
        [rows x heads x hd], rows_per_seq rows of each sequence in turn; k_prefix
        and v_prefix [kv_heads x P x hd]; k_tail and v_tail [slots x kv_heads x
        capacity x hd], sequence s's in slot slots[s] (None: slot s).  Row r
        attends the prefix and the first lens[r] positions of its tail (at most
        max_tail, by default the capacity; negative: the row is left out and
        its output is zero).  include/myl_hip.h states the arithmetic."""
        what = "attention_prefix_dev"
        if (score_shift | lut_shift | prob_frac) >> 8:
            _need_bytes(what, score_shift=score_shift, lut_shift=lut_shift, prob_frac=prob_frac)
        if not -2**63 <= score_mult < 2**63:
            raise ValueError(f"{what}: score_mult must be an int64, not {score_mult}")
        R, H, hd = q.shape
        KH, P = k_prefix.shape[:2]
        S, _, T = k_tail.shape[:3]
        dev = q.device
        if rows_per_seq <= 0 or R % rows_per_seq:
            raise ValueError(f"{what}: rows must be a multiple of rows_per_seq")
        if not (k_prefix.shape == v_prefix.shape == (KH, P, hd) and k_tail.shape == v_tail.shape == (S, KH, T, hd)):
            raise ValueError(f"{what}: prefix [kv_heads x P x hd], tails [slots x kv_heads x capacity x hd]")
        if max_tail is not None and not 0 <= max_tail <= T:
            raise ValueError(f"{what}: max_tail is at most the tails' capacity")
        _need_dev(what, dev, q=(q, "int16", None), k_prefix=(k_prefix, "int16", None), v_prefix=(v_prefix, "int16", None),
                  k_tail=(k_tail, "int16", None), v_tail=(v_tail, "int16", None), lens=(lens, "int32", (R,)),
                  exp_lut=(exp_lut, "int16", (exp_lut.numel(),)))
        n_seqs = R // rows_per_seq
        if slots is not None:
            _need_dev(what, dev, slots=(slots, "int32", (n_seqs,)))
        else:
            if not (S >= n_seqs):
                raise ValueError(f"{what}: fewer tails than sequences")
        stream = self._other_stream(dev) if out is None or workspace is None else None
        if out is None:
            out = self._empty((R, H, hd), "int16", dev, stream)
        _need_dev(what, dev, out=(out, "int16", None))
        if out.shape != q.shape:
            raise ValueError(f"{what}: out must have q's shape")

        def rows_of(t, name):
            row, head, one = _strides(t)
            if head not in (None, hd) or one not in (None, 1):
                raise ValueError(f"{what}: the heads of a row of {name} follow one another")
            return _apart(what, name, row, H * hd)

        ps, ts = _strides(k_prefix), _strides(k_tail)
        if not (ps[1] in (None, hd) and ps[2] in (None, 1) and ts[2] in (None, hd) and ts[3] in (None, 1)):
            raise ValueError(f"{what}: the positions of a KV head follow one another")
        if (k_prefix.stride() != v_prefix.stride() and ps != _strides(v_prefix)) or \
                (k_tail.stride() != v_tail.stride() and ts != _strides(v_tail)):
            raise ValueError(f"{what}: keys and values have the same strides")
        p_head, t_head = _apart(what, "prefix", ps[0], P * hd), _apart(what, "tails", ts[1], T * hd)
        t_slot = KH * T * hd if ts[0] is None else ts[0]  # 0: the slots share one tail
        max_tail = T if max_tail is None else max_tail
        ldq, ldo = rows_of(q, "q"), rows_of(out, "out")
        self._need_here(what, dev)
        ws = self._workspace(dev, workspace, stream, lib().myl_attention_prefix_workspace, n_seqs, rows_per_seq, H, KH, hd, P, max_tail)
        if stream is not None:
            self._after_last_use(what, dev, stream)
        rc = lib().myl_attention_prefix_dev(
            self._h, q.data_ptr(), n_seqs, rows_per_seq, ldq, H, KH, hd, k_prefix.data_ptr(), v_prefix.data_ptr(),
            P, p_head, k_tail.data_ptr(), v_tail.data_ptr(), S, t_slot, t_head, max_tail,
            None if slots is None else slots.data_ptr(), lens.data_ptr(), score_mult, score_shift, exp_lut.data_ptr(),
            exp_lut.numel(), lut_shift, prob_frac, out.data_ptr(), ldo, ws.data_ptr(),
            ws.numel() * ws.element_size())
        if rc:
            self.check(rc, what)
        return out

    def verify_drafts_workspace(self, target, exp_lut=None, draft=None):
        """A workspace for verify_drafts_dev on operands of these shapes, and on smaller ones."""
        n = lib().myl_verify_drafts_workspace(self._h, target.shape[0], target.shape[1] - 1, target.shape[2],
                                              0 if exp_lut is None else exp_lut.numel())
        return self._new_workspace(n, target.device, "verify_drafts_dev")

    def verify_drafts_dev(self, target, tokens, randoms, exp_lut=None, draft=None, n_draft=None, accepted=None, out=None,
                          workspace=None):
        """Drafted tokens against the target's probabilities: target int32
        [B x k+1 x V] logits, tokens int64 [B x k], randoms uint64 [B x k+1]
        (torch int64 tensors hold the bits), draft int32 [B x k x V] logits or
        None (drafts without probabilities), n_draft int32 [B] or None (k each);
        exp_lut None checks greedily (randoms may be None).  Drafts that were not
        drawn from the weights of `draft` (as this call draws with k = 0) are
        handed over without it: their tokens would be biased.  Returns (accepted
        int32 [B], out int64 [B x k+1]: accepted drafts, the next token, -1).
        include/myl_hip.h states the arithmetic."""
        what = "verify_drafts_dev"
        B, k1, V = target.shape
        dev, k = target.device, k1 - 1
        if k < 0:
            raise ValueError(f"{what}: target must be [B x k+1 x V]")
        _need_dev(what, dev, target=(target, "int32", None), tokens=(tokens, "int64", (B, k)))

        def rows_of(t, name, n):
            seq, row, one = _strides(t)
            if one not in (None, 1) or (None not in (seq, row) and seq != n * row):
                raise ValueError(f"{what}: the rows of {name} are evenly spaced")
            return _apart(what, name, seq if row is None else row, V)

        if exp_lut is not None:
            if randoms is None:
                raise ValueError(f"{what}: random numbers are needed unless the check is greedy")
            _need_dev(what, dev, exp_lut=(exp_lut, "int16", (exp_lut.numel(),)), randoms=(randoms, "int64", (B, k1)))
            if not exp_lut.numel():  # it has no address: the call would be the greedy one
                raise ValueError(f"{what}: the exp table must hold 1 to 32768 entries")
        if draft is not None:
            if draft.shape != (B, k, V):
                raise ValueError(f"{what}: draft must be [B x k x V]")
            _need_dev(what, dev, draft=(draft, "int32", None))
        if n_draft is not None:
            _need_dev(what, dev, n_draft=(n_draft, "int32", (B,)))
        stream = self._other_stream(dev) if accepted is None or out is None or workspace is None else None
        if accepted is None:
            accepted = self._empty(B, "int32", dev, stream)
        if out is None:
            out = self._empty((B, k1), "int64", dev, stream)
        _need_dev(what, dev, accepted=(accepted, "int32", (B,)), out=(out, "int64", (B, k1)))
        lut_len = 0 if exp_lut is None else exp_lut.numel()
        ldt, ldd = rows_of(target, "target", k1), V if draft is None or k == 0 else rows_of(draft, "draft", k)
        self._need_here(what, dev)
        ws = self._workspace(dev, workspace, stream, lib().myl_verify_drafts_workspace, B, k, V, lut_len)
        if stream is not None:
            self._after_last_use(what, dev, stream)
        rc = lib().myl_verify_drafts_dev(
            self._h, target.data_ptr(), ldt, None if draft is None or k == 0 else draft.data_ptr(), ldd, B, k, V, tokens.data_ptr(),
            None if n_draft is None else n_draft.data_ptr(), None if randoms is None else randoms.data_ptr(),
            None if exp_lut is None else exp_lut.data_ptr(), lut_len, accepted.data_ptr(), out.data_ptr(), ws.data_ptr(),
            ws.numel() * ws.element_size())
        if rc:
            self.check(rc, what)
        return accepted, out
