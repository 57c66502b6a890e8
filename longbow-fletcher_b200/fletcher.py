"""Python host binding of libcuda_fletcher.so (ctypes), mirroring the reference's Go device
interface for the embedding forward pass.

    Routing  : rows sent to experts (Cuda_Routing_*), their grouped products and the weighted sum;
               no counterpart in the reference
    Backend  ~ device.Backend  (internal/device/device.go:137-162)
    Tensor   ~ device.Tensor   (internal/device/device.go:5-117), the methods the hot path uses
    BertModel~ model.BertModel (internal/embeddings/model/bert.go:77-169) on the device

Every method calls the C ABI declared in include/fletcher_cuda.h; there is no CPU fallback:
if the library or a GPU is missing, construction raises.  Errors from the library raise
FletcherError carrying the library's message, the way the reference's Go wrapper panics
(cuda_linux.go:28-30).
"""
from __future__ import annotations

import ctypes
import os

import numpy as np

import synth

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libcuda_fletcher.so")

F32, F16, BF16 = 0, 1, 2
ACT_IDENTITY, ACT_GELU, ACT_TANH, ACT_SOFTMAX, ACT_SWIGLU = 0, 1, 2, 3, 4
POOL_CLS_TANH, POOL_MEAN_L2 = 0, 1
HALF_REFERENCE, HALF_RNE = 0, 1
SCORE_SOFTMAX, SCORE_SIGMOID = 0, 1
ROWS_TOKENS, ROWS_SLOTS = 0, 1
NORM_NONE, NORM_LAYER, NORM_RMS = 0, 1, 2
DTYPES = {"f32": F32, "f16": F16, "bf16": BF16}
_NP = {F32: np.float32, F16: np.float16}

_lib = None


class FletcherError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(f"[{code}] {msg}")
        self.code = code


def _sig(L):
    vp, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
    i32p, i64p = ctypes.POINTER(ctypes.c_int32), ctypes.POINTER(ctypes.c_int64)
    f32p = ctypes.POINTER(ctypes.c_float)
    sigs = {
        "Cuda_Init": (vp, []),
        "Cuda_GetDeviceCount": (i32, []),
        "Cuda_SetDevice": (i32, [vp, i32]),
        "Cuda_FreeContext": (None, [vp]),
        "Cuda_GetLastError": (i32, [vp, ctypes.c_char_p, i32]),
        "Cuda_Synchronize": (i32, [vp]),
        "Cuda_GetStream": (vp, [vp]),
        "Cuda_MemGetInfo": (i32, [vp, i64p, i64p]),
        "Cuda_Alloc": (vp, [vp, i64]),
        "Cuda_AllocTensor": (vp, [vp, i64, i64, i32]),
        "Cuda_WrapTensor": (vp, [vp, vp, i64, i64, i32]),
        "Cuda_FreeBuffer": (i32, [vp, vp]),
        "Cuda_CopyToDevice": (i32, [vp, i64, vp, i64]),
        "Cuda_CopyToHost": (i32, [vp, i64, vp, i64]),
        "Cuda_GetBufferContents": (vp, [vp]),
        "Cuda_BufferInfo": (i32, [vp, i64p, i64p, i32p]),
        "Cuda_CopyFromFloat32": (i32, [vp, f32p, i64]),
        "Cuda_ToHostFloat32": (i32, [vp, f32p, i64]),
        "Cuda_Linear_Fused": (i32, [vp, vp, i64, i64, vp, i64, vp, vp, i32]),
        "Cuda_LayerNorm": (i32, [vp, vp, vp, vp, vp, i64, i64, f32]),
        "Cuda_AddLayerNorm": (i32, [vp, vp, vp, vp, vp, i64, i64, f32]),
        "Cuda_Softmax": (i32, [vp, vp, vp, i64, i64]),
        "Cuda_Gather": (i32, [vp, vp, i32p, vp, i64, i64]),
        "Cuda_Add": (i32, [vp, vp, vp, i64]),
        "Cuda_Scale": (i32, [vp, vp, f32, i64]),
        "Cuda_AddScalar": (i32, [vp, vp, f32, i64]),
        "Cuda_AddBias": (i32, [vp, vp, vp, i64, i64]),
        "Cuda_Activation": (i32, [vp, vp, i64, i64, i32]),
        "Cuda_Cast": (i32, [vp, vp, vp, i64]),
        "Cuda_HasNaN": (i32, [vp, vp, i64, i32p]),
        "Cuda_Attention_Fused": (i32, [vp, vp, vp, vp, vp, i64, i64, i64, i32, f32]),
        "Cuda_Attention_VarLen": (i32, [vp, vp, vp, vp, vp, i32p, i32, i64, i32, f32]),
        "Cuda_Attention_VarLen_NoAlloc": (i32, [vp, vp, vp, vp, vp, i32p, i32, i64, i32, f32]),
        "Cuda_ApplyRoPE": (i32, [vp, vp, i64, i64, i32, i32]),
        "Cuda_ApplyRoPE_VarLen": (i32, [vp, vp, i32p, i32, i32, i32, f32]),
        "Cuda_MeanPoolL2": (i32, [vp, vp, i32p, i32, i64, vp]),
        "Cuda_Routing_Create": (i32, [vp, i64, i32, i32, ctypes.POINTER(vp)]),
        "Cuda_Routing_Free": (i32, [vp]),
        "Cuda_Routing_TopK": (i32, [vp, vp, i64, i32, i32, f32]),
        "Cuda_Routing_Assign": (i32, [vp, i32p, f32p, i64]),
        "Cuda_Routing_Read": (i32, [vp, i32p, f32p, i32p, i32p]),
        "Cuda_Routing_DevicePointers": (i32, [vp] + 4 * [ctypes.POINTER(vp)]),
        "Cuda_Linear_Grouped": (i32, [vp, vp, i32, i64, vp, i64, vp, vp, i32]),
        "Cuda_BlockNorm": (i32, [vp, vp, i64, i64, vp, vp, vp]),
        "Cuda_Combine_Grouped": (i32, [vp, vp, i64, vp, vp, vp]),
        "Cuda_Model_Create": (i32, [vp, vp, i32, ctypes.POINTER(vp)]),
        "Cuda_Model_LoadRaw": (i32, [vp, f32p, i64]),
        "Cuda_Model_WeightCount": (i64, [vp]),
        "Cuda_Model_ForwardBatch": (i32, [vp, i32p, i32p, i32, i32, f32p]),
        "Cuda_Model_ForwardBatchDevice": (i32, [vp, vp, i32p, i32, i32, vp]),
        "Cuda_Model_ForwardBatchEx": (i32, [vp, i32p, i32p, i32, i32, i32, vp]),
        "Cuda_Model_ForwardBatchAsync": (i32, [vp, vp, i32p, i32, i32, i32, vp, i64p]),
        "Cuda_Model_Wait": (i32, [vp, i64]),
        "Cuda_HostAlloc": (vp, [vp, i64]),
        "Cuda_HostFree": (None, [vp, vp]),
        "Cuda_Model_LastHidden": (i32, [vp, f32p, i64]),
        "Cuda_Model_SetStageTiming": (i32, [vp, i32]),
        "Cuda_Model_SetGraphs": (i32, [vp, i32]),
        "Cuda_Model_StageTimes": (i32, [vp, f32p, i64p, i32]),
        "Cuda_GetLaunchCount": (i64, [vp]),
        "Cuda_Debug_WaitTimeoutProbe": (i32, [vp, i64, i32]),
        "Cuda_Model_Free": (i32, [vp]),
        "Cuda_SetHalfConversion": (i32, [vp, i32]),
        "Cuda_Model_LoadTensor": (i32, [vp, ctypes.c_char_p, i32, vp, i64, i64, i32]),
        "Cuda_Model_TensorCount": (i32, [vp]),
        "Cuda_Model_TensorName": (i32, [vp, i32, ctypes.c_char_p, i32]),
        "Cuda_Model_IsLoaded": (i32, [vp]),
        "Cuda_Model_SetKeepHidden": (i32, [vp, i32]),
        "Cuda_At": (i32, [vp, i64, i64, f32p]),
        "Cuda_Set": (i32, [vp, i64, i64, f32]),
        "Cuda_Copy": (i32, [vp, vp, i64, vp, i64, i64]),
        "Cuda_Slice": (i32, [vp, vp, i64, i64, i64, i64, vp]),
        "Cuda_Mul": (i32, [vp, vp, i32, vp, i32, vp, i64, i64, i64]),
        "Cuda_Embedder_Create": (i32, [ctypes.POINTER(vp), i32, i32, i32, i64, ctypes.POINTER(vp)]),
        "Cuda_Embedder_CreateFake": (i32, [i32, i32, i64, i32, i64, ctypes.POINTER(vp)]),
        "Cuda_Embedder_Embed": (i32, [vp, i32p, i32p, i32, f32p]),
        "Cuda_Embedder_Throughput": (i32, [vp, ctypes.POINTER(ctypes.c_double), i32, i32]),
        "Cuda_Embedder_Counts": (i32, [vp, i64p, i64p, i32]),
        "Cuda_Embedder_Hidden": (i32, [vp]),
        "Cuda_Embedder_MaxBatch": (i32, [vp, i32p, i64p]),
        "Cuda_Embedder_LastError": (i32, [vp, ctypes.c_char_p, i32]),
        "Cuda_Embedder_Destroy": (None, [vp]),
        "Cuda_Server_Create": (i32, [vp, i32, i32, ctypes.POINTER(vp)]),
        "Cuda_Server_Submit": (i32, [vp, i32, i32p, i32p, i64p, i64p, f32p, i64p]),
        "Cuda_Server_Clock": (i64, []),
        "Cuda_Server_Wait": (i32, [vp, i64, ctypes.c_double, i64p]),
        "Cuda_Server_Latencies": (i32, [vp, i64, i64, i64p]),
        "Cuda_Server_Drain": (i32, [vp]),
        "Cuda_Server_Stats": (i32, [vp, vp]),
        "Cuda_Server_Destroy": (None, [vp]),
        "Cuda_Runtime_SplitByWeight": (i32, [i32p, i32, ctypes.POINTER(ctypes.c_double), i32, i32p]),
        "Cuda_Runtime_DynamicBatches": (i32, [i32p, i32, i32, i64, i32p, i32]),
    }
    for name, (res, args) in sigs.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    return L


def lib():
    """Loads the in-tree library (built by longbow-fletcher_b200/build.py)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FletcherError(-1, f"{LIB_PATH} is missing; run longbow-fletcher_b200/build.py")
        _lib = _sig(ctypes.CDLL(LIB_PATH))
    return _lib


def _i32p(a):
    return a.ctypes.data_as(ctypes.POINTER(ctypes.c_int32))


def _f32p(a):
    return a.ctypes.data_as(ctypes.POINTER(ctypes.c_float))


class PinnedArray:
    """Page-locked host array (Cuda_HostAlloc) viewed as numpy; freed with close()."""

    def __init__(self, be, shape, dtype):
        self.be = be
        self.dtype = np.dtype(dtype)
        n = int(np.prod(shape)) * self.dtype.itemsize
        self.ptr = lib().Cuda_HostAlloc(be.ctx, max(n, 1))
        if not self.ptr:
            be.check(3)  # FLETCHER_ERR_OOM
        buf = (ctypes.c_uint8 * max(n, 1)).from_address(self.ptr)
        self.array = np.frombuffer(buf, dtype=self.dtype, count=int(np.prod(shape))).reshape(shape)

    def close(self):
        if self.ptr:
            self.array = None
            lib().Cuda_HostFree(self.be.ctx, self.ptr)
            self.ptr = None


class Backend:
    """device.Backend on one GPU (NewCudaBackend / SetDevice, embeddings.go:105-135)."""

    def __init__(self, device: int = 0, dtype: str = "f32"):
        L = lib()
        n = L.Cuda_GetDeviceCount()
        if n <= 0:
            raise FletcherError(-1, "no CUDA device")
        self.ctx = L.Cuda_Init()
        if not self.ctx:
            raise FletcherError(-1, "Cuda_Init failed")
        self.dtype = DTYPES[dtype] if isinstance(dtype, str) else dtype
        if device:
            self.check(L.Cuda_SetDevice(self.ctx, device))
        self.device = device

    def name(self):
        return "CUDA-B200"

    def check(self, rc):
        if rc != 0:
            buf = ctypes.create_string_buffer(1024)
            lib().Cuda_GetLastError(self.ctx, buf, 1024)
            raise FletcherError(rc, buf.value.decode())
        return rc

    def new_tensor(self, r, c, data=None, dtype=None):
        return Tensor(self, r, c, self.dtype if dtype is None else dtype, data)

    def wrap(self, ptr, r, c, dtype=None):
        """A Tensor over (r, c) dense elements of device memory that the caller owns and keeps alive."""
        dt = self.dtype if dtype is None else dtype
        buf = lib().Cuda_WrapTensor(self.ctx, ctypes.c_void_p(ptr), r, c, dt)
        if not buf:
            self.check(1)  # FLETCHER_ERR_INVALID
        return Tensor(self, r, c, dt, buf=buf)

    def routing(self, max_rows, num_experts, top_k):
        return Routing(self, max_rows, num_experts, top_k)

    def synchronize(self):
        self.check(lib().Cuda_Synchronize(self.ctx))

    def device_count(self):
        return lib().Cuda_GetDeviceCount()

    def set_half_conversion(self, mode):
        """FLETCHER_HALF_REFERENCE (the reference's utils.go bytes, default) or FLETCHER_HALF_RNE."""
        self.check(lib().Cuda_SetHalfConversion(self.ctx, mode))

    def vram_usage(self):
        a, t = ctypes.c_int64(), ctypes.c_int64()
        self.check(lib().Cuda_MemGetInfo(self.ctx, ctypes.byref(a), ctypes.byref(t)))
        return a.value, t.value

    def stream(self):
        return lib().Cuda_GetStream(self.ctx)

    def launch_count(self):
        return lib().Cuda_GetLaunchCount(self.ctx)

    def close(self):
        if self.ctx:
            lib().Cuda_FreeContext(self.ctx)
            self.ctx = None


class Tensor:
    """device.Tensor: a dtype-tagged device buffer of (rows, cols).  T() returns a transposed
    view sharing the buffer (cpu_backend.go:306-314); only Mul reads the flag, as in the
    reference, where every other op sees the stored layout."""

    def __init__(self, be: Backend, r, c, dtype, data=None, buf=None):
        self.be, self.rows, self.cols, self.dtype = be, int(r), int(c), dtype
        self.trans = False
        self._owner = None
        self.buf = buf or lib().Cuda_AllocTensor(be.ctx, self.rows, self.cols, dtype)
        if not self.buf:
            be.check(3)
        if data is not None:
            self.copy_from_float32(data)

    def __del__(self):
        try:
            if self._owner is None and self.buf and self.be.ctx:
                lib().Cuda_FreeBuffer(self.be.ctx, self.buf)
        except Exception:
            pass

    def dims(self):
        return (self.cols, self.rows) if self.trans else (self.rows, self.cols)

    def T(self):
        v = Tensor.__new__(Tensor)
        v.be, v.rows, v.cols, v.dtype, v.buf = self.be, self.rows, self.cols, self.dtype, self.buf
        v.trans = not self.trans
        v._owner = self._owner or self  # keeps the buffer alive; the view never frees it
        return v

    def at(self, i, j):
        r = ctypes.c_float()
        self.be.check(lib().Cuda_At(self.buf, i, j, ctypes.byref(r)))
        return r.value

    def set(self, i, j, v):
        self.be.check(lib().Cuda_Set(self.buf, i, j, float(v)))

    def copy(self, other: "Tensor"):
        """device.Tensor.Copy: same dims, element-wise (cpu_backend.go:259-286)."""
        if self.dims() != other.dims():
            raise FletcherError(1, f"Copy: dimension mismatch {self.dims()} <- {other.dims()}")
        self.be.check(lib().Cuda_Copy(self.be.ctx, self.buf, 0, other.buf, 0, self.rows * self.cols))

    def slice(self, i, k, j, l):
        """device.Tensor.Slice: a new tensor holding a copy of [i:k, j:l] (cpu_backend.go:288-303)."""
        if k - i <= 0 or l - j <= 0:
            raise FletcherError(1, "Slice: invalid dimensions")
        out = Tensor(self.be, k - i, l - j, self.dtype)
        self.be.check(lib().Cuda_Slice(self.be.ctx, self.buf, i, k, j, l, out.buf))
        return out

    def mul(self, a: "Tensor", b: "Tensor"):
        """device.Tensor.Mul: self = a . b, honouring T() views (cpu_backend.go:316-372)."""
        ar, ac = a.dims()
        br, bc = b.dims()
        if ac != br:
            raise FletcherError(1, f"Mul: dimension mismatch a_cols={ac} b_rows={br}")
        if self.dims() != (ar, bc):
            raise FletcherError(1, f"Mul: result tensor dimension mismatch. Expected {ar}x{bc}, got {self.dims()}")
        self.be.check(lib().Cuda_Mul(self.be.ctx, a.buf, int(a.trans), b.buf, int(b.trans), self.buf, ar, bc, ac))

    def ptr(self):
        return lib().Cuda_GetBufferContents(self.buf)

    def copy_from_float32(self, data):
        a = np.ascontiguousarray(data, np.float32).reshape(-1)
        assert a.size == self.rows * self.cols
        self.be.check(lib().Cuda_CopyFromFloat32(self.buf, _f32p(a), a.size))

    def to_host(self):
        out = np.empty(self.rows * self.cols, np.float32)
        self.be.check(lib().Cuda_ToHostFloat32(self.buf, _f32p(out), out.size))
        return out.reshape(self.rows, self.cols)

    def raw_bytes(self):
        es = 4 if self.dtype == F32 else 2
        out = np.empty(self.rows * self.cols * es, np.uint8)
        self.be.check(lib().Cuda_CopyToHost(self.buf, 0, out.ctypes.data, out.size))
        return out

    # ---- ops (device.go:42-116)
    def linear(self, x: "Tensor", w: "Tensor", b: "Tensor | None", act=ACT_IDENTITY):
        n_out = w.cols // 2 if act == ACT_SWIGLU else w.cols
        y = Tensor(self.be, x.rows, n_out, x.dtype)
        self.be.check(lib().Cuda_Linear_Fused(self.be.ctx, x.buf, x.rows, x.cols, w.buf, w.cols,
                                              b.buf if b is not None else None, y.buf, act))
        return y

    def layer_norm(self, g, b, eps):
        self.be.check(lib().Cuda_LayerNorm(self.be.ctx, self.buf, g.buf, b.buf, self.buf, self.rows, self.cols, eps))

    def add_layer_norm(self, residual, g, b, eps):
        self.be.check(lib().Cuda_AddLayerNorm(self.be.ctx, self.buf, residual.buf, g.buf, b.buf,
                                              self.rows, self.cols, eps))

    def softmax(self):
        self.be.check(lib().Cuda_Softmax(self.be.ctx, self.buf, self.buf, self.rows, self.cols))

    def gather(self, indices):
        idx = np.ascontiguousarray(indices, np.int32)
        out = Tensor(self.be, idx.size, self.cols, self.dtype)
        self.be.check(lib().Cuda_Gather(self.be.ctx, self.buf, _i32p(idx), out.buf, idx.size, self.cols))
        return out

    def add(self, other):
        self.be.check(lib().Cuda_Add(self.be.ctx, self.buf, other.buf, self.rows * self.cols))

    def scale(self, v):
        self.be.check(lib().Cuda_Scale(self.be.ctx, self.buf, v, self.rows * self.cols))

    def add_scalar(self, v):
        self.be.check(lib().Cuda_AddScalar(self.be.ctx, self.buf, v, self.rows * self.cols))

    def add_bias(self, bias):
        self.be.check(lib().Cuda_AddBias(self.be.ctx, self.buf, bias.buf, self.rows, self.cols))

    def activation(self, act):
        self.be.check(lib().Cuda_Activation(self.be.ctx, self.buf, self.rows, self.cols, act))

    def cast(self, dtype):
        out = Tensor(self.be, self.rows, self.cols, dtype)
        self.be.check(lib().Cuda_Cast(self.be.ctx, self.buf, out.buf, self.rows * self.cols))
        return out

    def has_nan(self):
        r = ctypes.c_int32()
        self.be.check(lib().Cuda_HasNaN(self.be.ctx, self.buf, self.rows * self.cols, ctypes.byref(r)))
        return bool(r.value)

    def attention(self, q, k, v, batch, seq, heads, scale):
        out = Tensor(self.be, q.rows, q.cols, q.dtype)
        self.be.check(lib().Cuda_Attention_Fused(self.be.ctx, q.buf, k.buf, v.buf, out.buf, batch, seq, q.cols,
                                                 heads, scale))
        return out

    def attention_varlen(self, q, k, v, lengths, heads, scale):
        lens = np.ascontiguousarray(lengths, np.int32)
        out = Tensor(self.be, q.rows, q.cols, q.dtype)
        self.be.check(lib().Cuda_Attention_VarLen(self.be.ctx, q.buf, k.buf, v.buf, out.buf, _i32p(lens), lens.size,
                                                  q.cols, heads, scale))
        return out

    def apply_rope(self, batch, seq, heads, head_dim):
        self.be.check(lib().Cuda_ApplyRoPE(self.be.ctx, self.buf, batch, seq, heads, head_dim))

    def apply_rope_varlen(self, lengths, heads, head_dim, base):
        lens = np.ascontiguousarray(lengths, np.int32)
        self.be.check(lib().Cuda_ApplyRoPE_VarLen(self.be.ctx, self.buf, _i32p(lens), lens.size, heads, head_dim,
                                                  base))

    def block_norm(self, norm: "BlockNorm", out=None, out_norm=None):
        """Cuda_BlockNorm of this block output: (u, h), the residual stream and its norm.  The outputs
        may be given (this tensor and the residual among them); with neither, u is made, and h if
        there is a pre norm.  A tensor that is neither given nor made is None."""
        out, out_norm = norm._outputs(self, self.rows, out, out_norm)
        self.be.check(lib().Cuda_BlockNorm(self.be.ctx, self.buf, self.rows, self.cols, norm._ref(self.rows, self.cols),
                                           out.buf if out else None, out_norm.buf if out_norm else None))
        return out, out_norm

    def mean_pool_l2(self, lengths):
        lens = np.ascontiguousarray(lengths, np.int32)
        out = Tensor(self.be, lens.size, self.cols, F32)
        self.be.check(lib().Cuda_MeanPoolL2(self.be.ctx, self.buf, _i32p(lens), lens.size, self.cols, out.buf))
        return out


def _dense(t, cols, what):
    """Refuses a tensor whose rows are not `cols` wide; a flat one (one row or one column) holds them dense."""
    if t is not None and t.cols != cols and t.rows != 1 and t.cols != 1:
        raise FletcherError(1, f"{what} rows of {cols} columns, not {t.cols}")


class CBlockNorm(ctypes.Structure):
    """Matches FletcherBlockNorm in include/fletcher_cuda.h."""
    _fields_ = [("post_kind", ctypes.c_int32), ("pre_kind", ctypes.c_int32), ("eps", ctypes.c_float),
                ("residual_scale", ctypes.c_float), ("branch_scale", ctypes.c_float), ("reserved", ctypes.c_int32),
                ("gate_rows", ctypes.c_int64)] + [(n, ctypes.c_void_p) for n in (
                    "residual", "gate", "post_gamma", "post_beta", "pre_gamma", "pre_beta")]


class BlockNorm:
    """What happens to a block's output y (FletcherBlockNorm):
    u = residual_scale * residual + branch_scale * gate * post(y), h = pre(u)."""

    def __init__(self, post=NORM_NONE, pre=NORM_NONE, eps=1e-12, residual=None, gate=None, residual_scale=1.0,
                 branch_scale=1.0, post_gamma=None, post_beta=None, pre_gamma=None, pre_beta=None):
        self._tensors = dict(residual=residual, gate=gate, post_gamma=post_gamma, post_beta=post_beta,
                             pre_gamma=pre_gamma, pre_beta=pre_beta)  # kept alive with the handles
        self.c = CBlockNorm(post, pre, eps, residual_scale, branch_scale, 0, gate.rows if gate is not None else 0,
                            **{k: t.buf for k, t in self._tensors.items() if t is not None})
        self._p = ctypes.byref(self.c)
        self._residual_rows = residual.rows if residual is not None else float("inf")
        self._cols = [(n, t.cols) for n, t in (("residual", residual), ("gate", gate)) if hasattr(t, "cols")]

    def _ref(self, rows, cols=None):
        if self._residual_rows < rows:
            raise FletcherError(1, f"BlockNorm: the residual has {self._residual_rows} rows, {rows} are needed")
        for name, c in self._cols:
            if c != cols and cols is not None:
                raise FletcherError(1, f"BlockNorm: {name} must be of {cols} columns, not {c}")
        return self._p

    def _outputs(self, y, rows, out, out_norm, combine=False):
        _dense(out, y.cols, "BlockNorm: outputs must be")
        _dense(out_norm, y.cols, "BlockNorm: outputs must be")
        if out is None and out_norm is None:
            like = (self._tensors["residual"] or self._tensors["gate"] or y) if combine else y
            out = Tensor(y.be, rows, y.cols, like.dtype)
            if self.c.pre_kind != NORM_NONE:
                out_norm = Tensor(y.be, rows, y.cols, like.dtype)
        return out, out_norm


class Routing:
    """Rows sent to experts (Cuda_Routing_*): up to max_rows rows, top_k of num_experts each."""

    def __init__(self, be: Backend, max_rows, num_experts, top_k):
        self.be, self.num_experts, self.top_k, self.rows = be, num_experts, top_k, 0
        h = ctypes.c_void_p()
        self.h = None
        be.check(lib().Cuda_Routing_Create(be.ctx, max_rows, num_experts, top_k, ctypes.byref(h)))
        self.h = h

    def __del__(self):
        try:
            if self.h and self.be.ctx:
                lib().Cuda_Routing_Free(self.h)
        except Exception:
            pass

    def route(self, logits: Tensor, scoring=SCORE_SOFTMAX, normalise=True, scale=1.0):
        """Routes every row of logits (rows, num_experts) to its top_k largest."""
        if logits.cols != self.num_experts:
            raise FletcherError(1, f"Routing: logits have {logits.cols} columns for {self.num_experts} experts")
        self.be.check(lib().Cuda_Routing_TopK(self.h, logits.buf, logits.rows, scoring, int(normalise), scale))
        self.rows = logits.rows

    def assign(self, experts, weights=None):
        """Routes by given choices: host arrays (rows, top_k), -1 for none; weights default to 1."""
        e = np.ascontiguousarray(experts, np.int32).reshape(-1, self.top_k)
        w = None if weights is None else np.ascontiguousarray(weights, np.float32).reshape(-1, self.top_k)
        if w is not None and w.shape != e.shape:
            raise FletcherError(1, f"Routing: {w.shape} weights for {e.shape} choices")
        self.be.check(lib().Cuda_Routing_Assign(self.h, _i32p(e), None if w is None else _f32p(w), e.shape[0]))
        self.rows = e.shape[0]

    def read(self):
        """The last routing on the host: experts, weights, slots (rows, top_k) and offsets."""
        shape = (self.rows, self.top_k)
        e, s = np.empty(shape, np.int32), np.empty(shape, np.int32)
        w, o = np.empty(shape, np.float32), np.empty(self.num_experts + 1, np.int32)
        self.be.check(lib().Cuda_Routing_Read(self.h, _i32p(e), _f32p(w), _i32p(s), _i32p(o)))
        return {"experts": e, "weights": w, "slots": s, "offsets": o}

    def device_pointers(self):
        p = [ctypes.c_void_p() for _ in range(4)]
        self.be.check(lib().Cuda_Routing_DevicePointers(self.h, *(ctypes.byref(x) for x in p)))
        return dict(zip(("experts", "weights", "slots", "offsets"), (x.value for x in p)))

    def linear(self, x: Tensor, w: Tensor, b: "Tensor | None" = None, act=ACT_IDENTITY, grouped_input=False, out=None,
               dtype=None):
        """Cuda_Linear_Grouped: w (num_experts * in, out), b (num_experts, out); one output row a slot.
        x holds one row a token, or with grouped_input one row a slot.  The result has x's dtype, or F32."""
        if w.rows != self.num_experts * x.cols:
            raise FletcherError(1, f"Linear_Grouped: weight has {w.rows} rows, not {self.num_experts} x {x.cols}")
        cols = w.cols // 2 if act == ACT_SWIGLU else w.cols
        if act != ACT_SWIGLU or w.cols % 2 == 0:
            _dense(out, cols, "Linear_Grouped: result must hold")
        _dense(b, w.cols, "Linear_Grouped: bias must hold")
        y = out or Tensor(self.be, self.rows * self.top_k, cols, x.dtype if dtype is None else dtype)
        self.be.check(lib().Cuda_Linear_Grouped(self.h, x.buf, ROWS_SLOTS if grouped_input else ROWS_TOKENS, x.cols,
                                                w.buf, w.cols, b.buf if b is not None else None, y.buf, act))
        return y

    def combine(self, grouped: Tensor, norm: "BlockNorm | None" = None, out=None, out_norm=None):
        """Cuda_Combine_Grouped: the weighted sum of each row's slots, then the norm's u and h.
        Without a norm returns the sum, else (u, h) as Tensor.block_norm does; tensors that are made have
        the residual's dtype, else the gate's, else grouped's."""
        if norm is None:
            _dense(out, grouped.cols, "Combine_Grouped: outputs must be")
            out = out or Tensor(self.be, self.rows, grouped.cols, grouped.dtype)
            self.be.check(lib().Cuda_Combine_Grouped(self.h, grouped.buf, grouped.cols, None, out.buf, None))
            return out
        out, out_norm = norm._outputs(grouped, self.rows, out, out_norm, combine=True)
        self.be.check(lib().Cuda_Combine_Grouped(self.h, grouped.buf, grouped.cols, norm._ref(self.rows, grouped.cols),
                                                 out.buf if out else None, out_norm.buf if out_norm else None))
        return out, out_norm


class BertModel:
    """model.BertModel on the device (Cuda_Model_*): ForwardBatch(ids, lengths) -> [B, H]."""

    def __init__(self, be: Backend, cfg: synth.BertConfig, dtype=None):
        self.be, self.cfg = be, cfg
        self.dtype = be.dtype if dtype is None else (DTYPES[dtype] if isinstance(dtype, str) else dtype)
        self._c = synth.to_c(cfg)
        h = ctypes.c_void_p()
        be.check(lib().Cuda_Model_Create(be.ctx, ctypes.byref(self._c), self.dtype, ctypes.byref(h)))
        self.h = h

    def weight_count(self):
        return lib().Cuda_Model_WeightCount(ctypes.byref(self._c))

    def load_raw(self, blob):
        b = np.ascontiguousarray(blob, np.float32)
        self.be.check(lib().Cuda_Model_LoadRaw(self.h, _f32p(b), b.size))

    def load_tensor(self, name, array, dtype, transposed=False):
        """One checkpoint tensor by its reference name; `array` holds the raw values of `dtype`
        (float32, float16, or bfloat16 bit patterns as uint16), 1-D or 2-D."""
        a = np.ascontiguousarray(array)
        rows, cols = (1, a.size) if a.ndim <= 1 else (a.shape[0], int(np.prod(a.shape[1:])))
        self.be.check(lib().Cuda_Model_LoadTensor(self.h, name.encode(), dtype, a.ctypes.data, rows, cols,
                                                  int(transposed)))

    def is_loaded(self):
        return bool(lib().Cuda_Model_IsLoaded(self.h))

    def forward_batch(self, ids, lengths, pooling=POOL_MEAN_L2):
        ids = np.ascontiguousarray(ids, np.int32)
        lens = np.ascontiguousarray(lengths, np.int32)
        out = np.empty((lens.size, self.cfg.hidden), np.float32)
        self.be.check(lib().Cuda_Model_ForwardBatch(self.h, _i32p(ids), _i32p(lens), lens.size, pooling, _f32p(out)))
        return out

    def forward_batch_16(self, ids, lengths, pooling=POOL_MEAN_L2, out_dtype=F16):
        """Vectors as float16 (or bfloat16 bit patterns in uint16) — the fp16 transport."""
        ids = np.ascontiguousarray(ids, np.int32)
        lens = np.ascontiguousarray(lengths, np.int32)
        out = np.empty((lens.size, self.cfg.hidden), np.float16 if out_dtype == F16 else np.uint16)
        self.be.check(lib().Cuda_Model_ForwardBatchEx(self.h, _i32p(ids), _i32p(lens), lens.size, pooling, out_dtype,
                                                      out.ctypes.data))
        return out

    def forward_batch_async(self, ids_ptr, lengths, pooling, out_ptr, out_dtype=F32):
        """Enqueues a batch (ids and out: host pointers that stay valid until wait(ticket));
        returns its ticket.  The double-buffering half of the batcher loop."""
        lens = np.ascontiguousarray(lengths, np.int32)
        t = ctypes.c_int64()
        self.be.check(lib().Cuda_Model_ForwardBatchAsync(self.h, ctypes.c_void_p(ids_ptr), _i32p(lens), lens.size,
                                                         pooling, out_dtype, ctypes.c_void_p(out_ptr),
                                                         ctypes.byref(t)))
        return t.value

    def wait(self, ticket):
        self.be.check(lib().Cuda_Model_Wait(self.h, ticket))

    def forward_batch_device(self, d_ids_ptr, lengths, pooling, d_out_ptr):
        lens = np.ascontiguousarray(lengths, np.int32)
        self.be.check(lib().Cuda_Model_ForwardBatchDevice(self.h, ctypes.c_void_p(d_ids_ptr), _i32p(lens), lens.size,
                                                          pooling, ctypes.c_void_p(d_out_ptr)))

    STAGES = ["embed", "gemm_qkv", "rope", "attention", "gemm_o", "layernorm", "gemm_up", "activation",
              "gemm_down", "pool"]

    def set_keep_hidden(self, on: bool):
        self.be.check(lib().Cuda_Model_SetKeepHidden(self.h, int(on)))

    def set_graphs(self, on: bool):
        self.be.check(lib().Cuda_Model_SetGraphs(self.h, int(on)))

    def set_stage_timing(self, on: bool):
        self.be.check(lib().Cuda_Model_SetStageTiming(self.h, int(on)))

    def stage_times(self):
        """{stage: (milliseconds, timed calls)} since the last read."""
        n = len(self.STAGES)
        ms = np.zeros(n, np.float32)
        cnt = np.zeros(n, np.int64)
        self.be.check(lib().Cuda_Model_StageTimes(self.h, _f32p(ms), cnt.ctypes.data_as(ctypes.POINTER(ctypes.c_int64)), n))
        return {s: (float(ms[i]), int(cnt[i])) for i, s in enumerate(self.STAGES)}

    def last_hidden(self, T):
        out = np.empty((T, self.cfg.hidden), np.float32)
        self.be.check(lib().Cuda_Model_LastHidden(self.h, _f32p(out), out.size))
        return out

    def close(self):
        if self.h:
            lib().Cuda_Model_Free(self.h)
            self.h = None
