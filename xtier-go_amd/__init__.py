"""ctypes binding of libxtg_hip.so, the gfx950 kernel layer behind include/xtg_hip.h.

The binding is a thin mirror of the C ABI for tests, benchmarks and Python callers. It has no CPU fallback:
when the library is not built, every call raises.
"""
import ctypes
import json
import os

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
# XTG_HIP_LIB: another build of the same library (the phase-stamp build that `bench.py --gemv-phases` loads)
LIB_PATH = os.environ.get("XTG_HIP_LIB") or os.path.join(HERE, "libxtg_hip.so")

X_F32, X_BF16 = 0, 1
KV_BF16, KV_FP8, KV_NVFP4 = 0, 1, 2
LOGITS_NONE, LOGITS_LAST, LOGITS_ALL = 0, 1, 2   # xtg::Logits order (engine/include/xtg/model.h:28)

# Every function the header declares, with its ctypes signature: (name, restype, argtypes).
_P = ctypes.c_void_p
_I = ctypes.c_int
_SZ = ctypes.c_size_t
_ERR = [ctypes.c_char_p, _I]


class Nvfp4(ctypes.Structure):
    """xtg_nvfp4 (same fields as xtg::Nvfp4Weight, engine/include/xtg/kernels.h:13-20)."""
    _fields_ = [("codes", _P), ("scales", _P), ("glob", ctypes.c_float), ("n_out", _I), ("k", _I)]


class Bf16(ctypes.Structure):
    """xtg_bf16 (same fields as xtg::Bf16Weight, engine/include/xtg/kernels.h:22-25)."""
    _fields_ = [("data", _P), ("n_out", _I), ("k", _I)]


class Sampling(ctypes.Structure):
    """xtg_sampling (the fields of xtg::SamplingParams, engine/include/xtg/sampler.h:11-16)."""
    _fields_ = [("temperature", ctypes.c_float), ("top_p", ctypes.c_float), ("top_k", _I), ("min_p", ctypes.c_float)]


class AttnArgs(ctypes.Structure):
    """xtg_attn_args (the fields of xtg::AttnArgs, engine/include/xtg/kv.h:67-78)."""
    _fields_ = [("n_q", _I), ("pos0", ctypes.c_int64), ("heads", _I), ("kv_heads", _I), ("head_dim", _I),
                ("window", _I), ("scale", ctypes.c_float), ("q", _P), ("k", _P), ("v", _P), ("cache", _P),
                ("out", _P)]


class AttnExt(ctypes.Structure):
    """xtg_attn_ext."""
    _fields_ = [("n_q", _I), ("pos0", ctypes.c_int64), ("heads", _I), ("kv_heads", _I), ("head_dim", _I),
                ("window", _I), ("scale", ctypes.c_float), ("q", _P), ("k", _P), ("v", _P), ("cache", _P), ("out", _P),
                ("x_dtype", _I), ("softcap", ctypes.c_float), ("slopes", _P), ("first", _P), ("end", _P)]


_F = ctypes.c_float
_I64 = ctypes.c_int64


class PagedRowsArgs(ctypes.Structure):
    """xtg_paged_rows."""
    _fields_ = [("n_seqs", _I), ("n_rows", _I), ("pos", _P), ("starts", _P), ("pages", _P), ("max_pages", _I)]


class PagedAppendArgs(ctypes.Structure):
    """xtg_paged_append."""
    _fields_ = [("heads", _I), ("q", _P), ("q_out", _P), ("k", _P), ("v", _P), ("q_stride", _I64), ("k_stride", _I64),
                ("v_stride", _I64), ("x_dtype", _I), ("theta", _F), ("norm", _I), ("qscale", _P)]


class PagedAttnArgs(ctypes.Structure):
    """xtg_paged_attn."""
    _fields_ = [("heads", _I), ("q", _P), ("q_stride", _I64), ("out", _P), ("x_dtype", _I), ("window", _I), ("scale", _F),
                ("softcap", _F)]


class DoryConfig(ctypes.Structure):
    """xtg_dory_config."""
    _fields_ = [(n, _I) for n in ("hidden", "ffn", "heads", "kv_heads", "head_dim", "vocab", "n_in", "n_rec", "n_out",
                                  "loops", "window", "ring_slots")] + \
               [("context", _I64), ("theta_sliding", _F), ("theta_full", _F), ("kv_dtype", _I), ("kv_mode", _I)]


class DoryLayer(ctypes.Structure):
    """xtg_dory_layer."""
    _fields_ = [("kind", _I)] + [(n, Nvfp4) for n in ("q", "k", "v", "g", "o", "gate", "up", "down")] + \
               [(n, _P) for n in ("qscale", "gscale", "sg", "su", "lr")]


SIGNATURES = [
    ("xtg_hip_open", _P, [ctypes.c_char_p] + _ERR),
    ("xtg_hip_close", None, [_P]),
    ("xtg_hip_info", _I, [_P, ctypes.c_char_p, _I]),
    ("xtg_hip_stream", _P, [_P]),
    ("xtg_hip_prepare_nvfp4", _I, [_P, ctypes.POINTER(Nvfp4)] + _ERR),
    ("xtg_hip_release_nvfp4", _I, [_P, _P] + _ERR),
    ("xtg_hip_matmul_nvfp4", _I, [_P, ctypes.POINTER(Nvfp4), _I, _P, _I, ctypes.POINTER(_P)] + _ERR),
    ("xtg_hip_matmul_nvfp4_dev", _I, [_P, ctypes.POINTER(Nvfp4), _I, _P, _I, _I, _P, _SZ] + _ERR),
    ("xtg_hip_prepare_bf16", _I, [_P, ctypes.POINTER(Bf16)] + _ERR),
    ("xtg_hip_release_bf16", _I, [_P, _P] + _ERR),
    ("xtg_hip_matmul_bf16", _I, [_P, ctypes.POINTER(Bf16), _P, _I, _P] + _ERR),
    ("xtg_hip_matmul_bf16_dev", _I, [_P, ctypes.POINTER(Bf16), _P, _I, _I, _P, _SZ] + _ERR),
    ("xtg_hip_kv_create", _P, [_P, _I, _I, _I64, _I, _I] + _ERR),
    ("xtg_hip_kv_destroy", None, [_P, _P]),
    ("xtg_hip_kv_store", _I, [_P, _P, _I64, _I, _P, _P] + _ERR),
    ("xtg_hip_kv_globals", _I, [_P, _P, _F, _F] + _ERR),
    ("xtg_hip_kv_write", _I, [_P, _P, _I64, _I, _P, _P, _I] + _ERR),
    ("xtg_hip_kv_read", _I, [_P, _P, _I64, _I, _P, _P, _I] + _ERR),
    ("xtg_hip_kv_load", _I, [_P, _P, _I, _I64, _I64, _P, _P] + _ERR),
    ("xtg_hip_kv_bytes", _I64, [_P, _P]),
    ("xtg_hip_kv_save", _I, [_P, _P, _P, _SZ] + _ERR),
    ("xtg_hip_kv_restore", _I, [_P, _P, _P, _SZ] + _ERR),
    ("xtg_hip_kv_copy", _I, [_P, _P, _P] + _ERR),
    ("xtg_hip_nvfp4_tiles", _I, [_P, _P, _P, _SZ] + _ERR),
    ("xtg_hip_kv_release", _I, [_P, _P] + _ERR),
    ("xtg_hip_attention", _I, [_P, ctypes.POINTER(AttnArgs)] + _ERR),
    ("xtg_hip_attention_noalloc", _I, [_P, ctypes.POINTER(AttnArgs)] + _ERR),
    ("xtg_hip_attention_ext", _I, [_P, ctypes.POINTER(AttnExt)] + _ERR),
    ("xtg_hip_paged_create", _P, [_P, _I, _I, _I64, _I, _I] + _ERR),
    ("xtg_hip_paged_destroy", None, [_P, _P]),
    ("xtg_hip_paged_globals", _I, [_P, _P, _F, _F] + _ERR),
    ("xtg_hip_paged_append", _I, [_P, _P, ctypes.POINTER(PagedRowsArgs), ctypes.POINTER(PagedAppendArgs)] + _ERR),
    ("xtg_hip_paged_read", _I, [_P, _P, ctypes.POINTER(PagedRowsArgs), _P, _P, _I] + _ERR),
    ("xtg_hip_paged_attention", _I, [_P, _P, ctypes.POINTER(PagedRowsArgs), ctypes.POINTER(PagedAttnArgs)] + _ERR),
    ("xtg_hip_qk_rope_norm", _I, [_P, _P, _P, _I, _I, _I, _I, _I64, _F, _P] + _ERR),
    ("xtg_hip_slerp_residual", _I, [_P, _P, _P, _P, _I, _I] + _ERR),
    ("xtg_hip_swiglu_norm", _I, [_P, _P, _P, _P, _P, _I, _I] + _ERR),
    ("xtg_hip_gate_norm", _I, [_P, _P, _P, _P, _I, _I] + _ERR),
    ("xtg_hip_add_norm", _I, [_P, _P, _P, _P, _I, _I] + _ERR),
    ("xtg_hip_argmax", _I, [_P, _P, _I, _I, _P] + _ERR),
    ("xtg_hip_sample", _I, [_P, _P, _I, _I, ctypes.POINTER(Sampling), _P, _P] + _ERR),
    ("xtg_hip_dory_create", _P, [_P, ctypes.POINTER(DoryConfig), ctypes.POINTER(DoryLayer), ctypes.POINTER(Nvfp4),
                                 _P] + _ERR),
    ("xtg_hip_dory_destroy", None, [_P]),
    ("xtg_hip_dory_head_bf16", _I, [_P, ctypes.POINTER(Bf16)] + _ERR),
    ("xtg_hip_dory_forward", _I, [_P, _P, _I, _I64, _P] + _ERR),
    ("xtg_hip_dory_prefill", _I, [_P, _P, _I, _I64, _I, _P] + _ERR),
    ("xtg_hip_dory_cache", _P, [_P, _I, _I]),
    ("xtg_hip_dory_snapshot", _I, [_P, _I] + _ERR),
    ("xtg_hip_dory_restore", _I, [_P, _I] + _ERR),
    ("xtg_hip_x_operand_bytes", _SZ, [_I]),
    ("xtg_hip_prep_x", _I, [_P, _P, _I, _I, _I, _P] + _ERR),
    ("xtg_hip_matmul_nvfp4_op", _I, [_P, ctypes.POINTER(Nvfp4), _I, _P, _I, _P, _SZ] + _ERR),
    ("xtg_hip_alloc", _I, [_P, _SZ, ctypes.POINTER(_P)] + _ERR),
    ("xtg_hip_release", None, [_P, _P]),
    ("xtg_hip_write", _I, [_P, _P, _SZ, _P, _SZ] + _ERR),
    ("xtg_hip_read", _I, [_P, _P, _SZ, _P, _SZ] + _ERR),
    ("xtg_hip_copy", _I, [_P, _P, _SZ, _P, _SZ, _SZ] + _ERR),
    ("xtg_hip_finish", _I, [_P] + _ERR),
    ("xtg_hip_graph_begin", _I, [_P] + _ERR),
    ("xtg_hip_graph_end", _I, [_P, ctypes.c_char_p, ctypes.POINTER(_P)] + _ERR),
    ("xtg_hip_graph_launch", _I, [_P, _P] + _ERR),
    ("xtg_hip_graph_destroy", None, [_P, _P]),
    ("xtg_hip_read_probe_partials", _SZ, [_SZ]),
    ("xtg_hip_read_probe", _I, [_P, _P, _SZ, _P] + _ERR),
    ("xtg_hip_profile", _I, [_P, _I] + _ERR),
    ("xtg_hip_profile_report", _I, [_P, ctypes.c_char_p, _I]),
]

_lib = None


class XtgError(RuntimeError):
    pass


def lib():
    """The loaded library; raises when it is not built (there is no fallback path)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise XtgError("libxtg_hip.so is not built (run __graft_entry__.build() or xtier-go_amd/build.py)")
        l = ctypes.CDLL(LIB_PATH)
        for name, res, args in SIGNATURES:
            f = getattr(l, name)
            f.restype = res
            f.argtypes = args
        _lib = l
    return _lib


_ERR_LEN = 2048
_ErrBuf = ctypes.c_char * _ERR_LEN


def _errbuf():
    return _ErrBuf()


def _check(rc, err):
    if rc != 0:
        raise XtgError(err.value.decode(errors="replace"))


def _ptr(a):
    """Address of a numpy array or a torch tensor (device or host), or an int."""
    if a is None:
        return None
    if isinstance(a, int):
        return a
    if isinstance(a, np.ndarray):
        return a.ctypes.data
    return a.data_ptr()   # torch.Tensor


# What elements an array holds: X_F32, X_BF16 (as 16-bit integers too, which is how numpy holds them) or _I32. Tensors'
# dtypes are torch's own objects, looked up by name once.
_I32 = -2
_KIND_OF = {"float32": X_F32, "bfloat16": X_BF16, "uint16": X_BF16, "int16": X_BF16, "int32": _I32}
_kinds = {}


def _device_ptr(b, name, a, n, kind):
    """Address of n elements of a kind in backend b's device memory. An array that is elsewhere, of another dtype, strided,
    too short or freed is refused: the kernels would read or write past it. An address (an int) or None is taken as it is."""
    if a is None:
        return None
    cls = a.__class__
    if cls is not DeviceArray and cls is not int:
        try:   # a torch tensor as it should be
            if _kinds[a.dtype] == kind and a.numel() >= n and a.is_contiguous() and a.get_device() == b.device:
                return a.data_ptr()
        except (AttributeError, KeyError):
            pass
    if isinstance(a, int):
        return a
    if isinstance(a, DeviceArray):
        at, size, here, whole = a.ptr if a.ptr and a.b.h else None, a.nbytes // a.dtype.itemsize, a.b.device == b.device, True
    elif hasattr(a, "get_device"):
        at, size, here, whole = a.data_ptr(), a.numel(), a.get_device() == b.device, a.is_contiguous()
    else:
        raise XtgError("%s is not in device memory" % name)
    if a.dtype not in _kinds:
        _kinds[a.dtype] = _KIND_OF.get(str(a.dtype).replace("torch.", ""))
    if _kinds[a.dtype] != kind:
        want = {X_F32: "row type FP32", X_BF16: "row type BF16", _I32: "int32"}.get(kind, "unknown row type %s" % kind)
        raise XtgError("%s is %s, not of the call's %s" % (name, a.dtype, want))
    if not here:
        raise XtgError("%s is not in the memory of the backend's device" % name)
    if not whole:
        raise XtgError("%s is not contiguous" % name)
    if size < n:
        raise XtgError("%s has %d elements, the call's rows of it take %d" % (name, size, n))
    if n > 0 and not at:
        raise XtgError("%s has been freed" % name)
    return at


def _device_rows(b, k, v, n, kind):
    """_device_ptr of a call's k and v, in one step where both are torch tensors as they should be."""
    try:
        if (_kinds[k.dtype] == kind and v.dtype is k.dtype and k.numel() >= n and v.numel() >= n and k.is_contiguous() and
                v.is_contiguous() and k.get_device() == v.get_device() == b.device):
            return k.data_ptr(), v.data_ptr()
    except (AttributeError, KeyError):
        pass
    return _device_ptr(b, "k", k, n, kind), _device_ptr(b, "v", v, n, kind)


def _rows_ptr(b, name, a, n, width, stride, kind):
    """_device_ptr of n rows of `width` elements, `stride` elements apart (0: packed). A tensor may be part of wider rows, as q,
    k and v of one projection are, where its rows are as far apart as the call says."""
    if not stride:
        return _device_ptr(b, name, a, n * width, kind)
    if n and hasattr(a, "stride") and not a.is_contiguous():
        at = _device_ptr(b, name, a[0], width, kind)   # a row of it
        if a.shape[0] < n:
            raise XtgError("%s has %d rows, the call %d" % (name, a.shape[0], n))
        if a.stride(0) != stride:
            raise XtgError("%s has rows %d elements apart, not the call's %d" % (name, a.stride(0), stride))
        return at
    return _device_ptr(b, name, a, (n - 1) * stride + width if n else 0, kind)


class _Address(int):
    """The address of an array, which it holds: with a second reference numpy refuses to resize (move) it in place. A copy
    or a pickle of it reads its own array's."""

    def __new__(cls, array):
        at = int.__new__(cls, array.ctypes.data)
        at.array = array
        return at

    def __reduce__(self):
        return _Address, (self.array,)


class _Array:
    """A Weight's array attribute: its address is read when the array is set, not on every call (numpy's .ctypes takes
    about 0.6 us, three times per weight of a call; a call of four projections spent half of its 14 us there)."""

    def __set_name__(self, owner, name):
        self.name, self.held = name, "_" + name

    def __get__(self, w, owner=None):
        if w is None:
            return self
        try:
            return w.__dict__[self.name]
        except KeyError:
            raise AttributeError(self.name) from None

    def __set__(self, w, a):
        w.__dict__[self.name] = a
        w.__dict__.pop(self.held, None)
        if hasattr(a, "ctypes"):
            w.__dict__[self.held] = _Address(a)

    def __delete__(self, w):
        self.__get__(w)
        del w.__dict__[self.name]
        w.__dict__.pop(self.held, None)


class Weight:
    """An NVFP4 weight held in host memory: codes [n][k/2] u8, scales [n][k/16] u8 (E4M3), global f32."""
    codes, scales = _Array(), _Array()

    def __init__(self, codes, scales, glob=1.0):
        self.codes = np.ascontiguousarray(codes, dtype=np.uint8)
        self.scales = np.ascontiguousarray(scales, dtype=np.uint8)
        self.glob = float(glob)
        self.n_out = self.codes.shape[0]
        self.k = self.codes.shape[1] * 2
        assert self.scales.shape == (self.n_out, self.k // 16)

    def struct(self):
        try:
            return Nvfp4(self._codes, self._scales, self.glob, self.n_out, self.k)
        except AttributeError:   # no addresses: restored from a state of codes and scales alone, or no arrays any more
            return Nvfp4(self.codes.ctypes.data, self.scales.ctypes.data, self.glob, self.n_out, self.k)


class HipBackend:
    """One xtg_hip handle (a device, its stream and prepared weights)."""

    def __init__(self, device=0):
        self.device = device
        err = _errbuf()
        self.h = lib().xtg_hip_open(json.dumps({"device": device}).encode(), err, len(err))
        if not self.h:
            raise XtgError(err.value.decode(errors="replace"))
        self._err = _errbuf()   # of the calls that a decode step makes for every layer (one thread at a time)
        # Prepared weights are keyed by the address of their codes (as in the reference); every Weight passed in
        # is kept alive here so that no later array can reuse an address that still names a prepared copy.
        self._weights = {}

    def close(self):
        if self.h:
            lib().xtg_hip_close(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def info(self):
        buf = ctypes.create_string_buffer(4096)
        n = lib().xtg_hip_info(self.h, buf, len(buf))
        if n < 0:
            raise XtgError("info failed")
        return json.loads(buf.value.decode())

    @property
    def stream(self):
        return lib().xtg_hip_stream(self.h)

    def _hold(self, ws):
        arr, held = (Nvfp4 * len(ws))(), self._weights
        try:
            for i, w in enumerate(ws):   # as Weight.struct, without a structure per weight
                at = w._codes
                arr[i] = at, w._scales, w.glob, w.n_out, w.k
                if at not in held:
                    held[int(at)] = w
        except AttributeError:
            for i, w in enumerate(ws):
                arr[i] = w.struct()
                held.setdefault(arr[i].codes, w)
        return arr

    def prepare(self, w):
        err = _errbuf()
        arr = self._hold([w])
        _check(lib().xtg_hip_prepare_nvfp4(self.h, arr, err, len(err)), err)

    def nvfp4_tiles(self, w):
        """The device tile layout prepared for w (uint8, ceil(n/16) * ceil(k/128) * 1152 bytes)."""
        n, k = w.codes.shape[0], w.codes.shape[1] * 2
        out = np.empty(((n + 15) // 16) * ((k + 127) // 128) * 1152, np.uint8)
        err = _errbuf()
        _check(lib().xtg_hip_nvfp4_tiles(self.h, w.codes.ctypes.data, out.ctypes.data, out.nbytes, err, len(err)), err)
        return out

    def release_weight(self, w):
        """Drop the device copy of w (and let its host arrays go)."""
        err = _errbuf()
        key = w.codes.ctypes.data
        _check(lib().xtg_hip_release_nvfp4(self.h, key, err, len(err)), err)
        self._weights.pop(key, None)

    def matmul(self, ws, x):
        """Host-synchronous matmul_nvfp4: x float32 [m][k] -> list of float32 [m][n_i]."""
        x = np.ascontiguousarray(x, dtype=np.float32)
        m = x.shape[0]
        ys = [np.empty((m, w.n_out), dtype=np.float32) for w in ws]
        yp = (_P * len(ws))(*[y.ctypes.data for y in ys])
        err = _errbuf()
        _check(lib().xtg_hip_matmul_nvfp4(self.h, self._hold(ws), len(ws), x.ctypes.data, m, yp, err, len(err)), err)
        return ys

    def matmul_dev(self, ws, x, x_dtype, m, y, y_offset=0):
        """Queued device matmul: x, y are device addresses (ints or torch tensors)."""
        err = _errbuf()
        _check(lib().xtg_hip_matmul_nvfp4_dev(self.h, self._hold(ws), len(ws), _ptr(x), x_dtype, m, _ptr(y), y_offset,
                                              err, len(err)), err)

    @staticmethod
    def x_operand_bytes(k):
        return lib().xtg_hip_x_operand_bytes(k)

    def prep_x(self, x, x_dtype, m, k, op):
        """Queued: the matrix-core operand of x ([m][k] on the device) into the device buffer op."""
        err = _errbuf()
        _check(lib().xtg_hip_prep_x(self.h, _ptr(x), x_dtype, m, k, _ptr(op), err, len(err)), err)

    def matmul_op(self, ws, op, m, y, y_offset=0):
        """Queued: the projections of a prepared operand into y (as matmul_dev)."""
        err = _errbuf()
        _check(lib().xtg_hip_matmul_nvfp4_op(self.h, self._hold(ws), len(ws), _ptr(op), m, _ptr(y), y_offset, err,
                                             len(err)), err)

    # ---- BF16 weights (xtg::Bf16Weight): w is a C-contiguous uint16 array [n_out][k] of BF16 bits
    def _bf16(self, w):
        assert w.dtype == np.uint16 and w.ndim == 2 and w.flags.c_contiguous
        self._weights.setdefault(w.ctypes.data, w)
        return Bf16(w.ctypes.data, w.shape[0], w.shape[1])

    def prepare_bf16(self, w):
        err = _errbuf()
        st = self._bf16(w)
        _check(lib().xtg_hip_prepare_bf16(self.h, ctypes.byref(st), err, len(err)), err)

    def release_bf16(self, w):
        err = _errbuf()
        _check(lib().xtg_hip_release_bf16(self.h, w.ctypes.data, err, len(err)), err)
        self._weights.pop(w.ctypes.data, None)

    def matmul_bf16(self, w, x):
        """Host-synchronous matmul_bf16: x float32 [m][k] -> float32 [m][n_out]."""
        x = np.ascontiguousarray(x, dtype=np.float32)
        y = np.empty((x.shape[0], w.shape[0]), dtype=np.float32)
        err = _errbuf()
        st = self._bf16(w)
        _check(lib().xtg_hip_matmul_bf16(self.h, ctypes.byref(st), x.ctypes.data, x.shape[0], y.ctypes.data, err,
                                         len(err)), err)
        return y

    def matmul_bf16_dev(self, w, x, x_dtype, m, y, y_offset=0):
        """Queued device matmul_bf16: x, y are device addresses."""
        err = _errbuf()
        st = self._bf16(w)
        _check(lib().xtg_hip_matmul_bf16_dev(self.h, ctypes.byref(st), _ptr(x), x_dtype, m, _ptr(y), y_offset, err,
                                             len(err)), err)

    def alloc(self, nbytes):
        err = _errbuf()
        out = _P()
        _check(lib().xtg_hip_alloc(self.h, nbytes, ctypes.byref(out), err, len(err)), err)
        return out.value

    def release(self, mem):
        lib().xtg_hip_release(self.h, mem)

    def write(self, mem, src, offset=0):
        src = np.ascontiguousarray(src)
        err = _errbuf()
        _check(lib().xtg_hip_write(self.h, _ptr(mem), offset, src.ctypes.data, src.nbytes, err, len(err)), err)

    def read(self, mem, dst, offset=0):
        err = _errbuf()
        _check(lib().xtg_hip_read(self.h, _ptr(mem), offset, dst.ctypes.data, dst.nbytes, err, len(err)), err)
        return dst

    def copy(self, src, dst, nbytes, src_offset=0, dst_offset=0):
        err = _errbuf()
        _check(lib().xtg_hip_copy(self.h, _ptr(src), src_offset, _ptr(dst), dst_offset, nbytes, err, len(err)), err)

    def finish(self):
        err = _errbuf()
        _check(lib().xtg_hip_finish(self.h, err, len(err)), err)

    def graph_begin(self):
        err = _errbuf()
        _check(lib().xtg_hip_graph_begin(self.h, err, len(err)), err)

    def graph_end(self, name=None):
        """The captured graph (an opaque handle for graph_launch / graph_destroy)."""
        err = _errbuf()
        g = _P()
        _check(lib().xtg_hip_graph_end(self.h, name.encode() if name else None, ctypes.byref(g), err, len(err)), err)
        return g.value

    def graph_launch(self, g):
        err = _errbuf()
        _check(lib().xtg_hip_graph_launch(self.h, g, err, len(err)), err)

    def graph_destroy(self, g):
        lib().xtg_hip_graph_destroy(self.h, g)

    def profile(self, enable=True, launches=False):
        """Per-kernel event timing on (launches: also every launch's time in queue order) or off."""
        err = _errbuf()
        _check(lib().xtg_hip_profile(self.h, (2 if launches else 1) if enable else 0, err, len(err)), err)

    def profile_report(self, launches=False):
        """{kernel name: {"calls": n, "ms": total}} since the last report (waits for queued work); with launches,
        also the list [(name, ms), ...] of every launch in queue order (profiling turned on with launches=True)."""
        buf = ctypes.create_string_buffer(1 << 22)
        n = lib().xtg_hip_profile_report(self.h, buf, len(buf))
        if n < 0 or n >= len(buf):
            raise XtgError("profile report failed")
        rep = json.loads(buf.value.decode())
        if launches:
            return rep["kernels"], [tuple(x) for x in rep.get("launches", [])]
        return rep["kernels"]

    def array(self, a=None, shape=None, dtype=np.float32):
        """A device buffer owned by this backend, filled from the numpy array a (or left unset)."""
        return DeviceArray(self, a, shape, dtype)

    # ---- KV caches and attention (engine/include/xtg/kv.h)
    def kv_cache(self, kv_heads, head_dim, slots, ring=0, dtype=KV_BF16):
        return KvCache(self, kv_heads, head_dim, slots, ring, dtype)

    def attention(self, cache, q, k, v, out, n_q, pos0, heads, window=0, scale=None):
        """Queued device attention: q, k, v, out device buffers as xtg::AttnArgs."""
        sc = float(np.float32(1) / np.sqrt(np.float32(cache.head_dim))) if scale is None else float(scale)
        a = AttnArgs(n_q, pos0, heads, cache.kv_heads, cache.head_dim, window, sc, _ptr(q), _ptr(k), _ptr(v), cache.h,
                     _ptr(out))
        err = _errbuf()
        _check(lib().xtg_hip_attention(self.h, ctypes.byref(a), err, len(err)), err)

    def attention_noalloc(self, cache, q, k, v, out, n_q, pos0, heads, window=0, scale=None):
        """The same call with its partials in the device's fixed scratch (xtg_hip_attention_noalloc)."""
        sc = float(np.float32(1) / np.sqrt(np.float32(cache.head_dim))) if scale is None else float(scale)
        a = AttnArgs(n_q, pos0, heads, cache.kv_heads, cache.head_dim, window, sc, _ptr(q), _ptr(k), _ptr(v), cache.h,
                     _ptr(out))
        err = _errbuf()
        _check(lib().xtg_hip_attention_noalloc(self.h, ctypes.byref(a), err, len(err)), err)

    def attention_ext(self, cache, q, k, v, out, n_q, pos0, heads, kv_heads, head_dim, x_dtype=X_F32, window=0,
                      scale=None, softcap=0.0, slopes=None, first=None, end=None):
        """Queued device attention with capped, biased and masked scores (xtg_hip_attention_ext) over a cache of any
        dtype (None: the call's own keys alone): row i, at t = pos0 + i, sees positions first[i] <= p < end[i] (None:
        from 0, to t) and p > t - window; scores softcap * tanh(scale * q.k / softcap) - slopes[head] * |t - p|. k and
        v None: the call's own rows are in the cache. q, k, v, out: device rows of x_dtype; slopes: device FP32
        [heads]; first, end: device int32 [n_q]."""
        sc = head_dim ** -0.5 if scale is None else scale
        if cache is not None and not cache.h:   # NULL would mean no cache
            raise XtgError("attention_ext: the cache has been destroyed")
        nq, nk = n_q * heads * head_dim, n_q * kv_heads * head_dim
        a = AttnExt(n_q, pos0, heads, kv_heads, head_dim, window, sc, _device_ptr(self, "q", q, nq, x_dtype),
                    _device_ptr(self, "k", k, nk, x_dtype), _device_ptr(self, "v", v, nk, x_dtype),
                    cache.h if cache is not None else None, _device_ptr(self, "out", out, nq, x_dtype), x_dtype, softcap,
                    _device_ptr(self, "slopes", slopes, heads, X_F32), _device_ptr(self, "first", first, n_q, _I32),
                    _device_ptr(self, "end", end, n_q, _I32))
        err = self._err
        _check(lib().xtg_hip_attention_ext(self.h, ctypes.byref(a), err, len(err)), err)

    # ---- paged caches
    def paged_cache(self, kv_heads, head_dim, pages, page_size=64, dtype=KV_BF16):
        """A pool of pages of page_size positions (a power of two from 32 to 4096) for many sequences."""
        return PagedCache(self, kv_heads, head_dim, pages, page_size, dtype)

    def paged_rows(self, pos, pages, n_rows=None, starts=None):
        """Whose the rows of a call are (xtg_paged_rows), for any number of calls on pools of the same pages: device int32
        pos [n_seqs], pages [n_seqs][max_pages] and, unless row s is sequence s's, starts [n_seqs + 1], with which n_rows
        says how many rows the call has."""
        return PagedRows(self, pos, pages, n_rows, starts)

    # ---- the Dory decode step
    def dory(self, weights):
        """A decode session over DoryWeights (xtier_go_amd.workloads); the weights stay referenced by it."""
        return DorySession(self, weights)

    # ---- row kernels (queued, device buffers)
    def qk_rope_norm(self, q, k, m, heads, kv_heads, head_dim, pos0, theta, qscale=None):
        err = _errbuf()
        _check(lib().xtg_hip_qk_rope_norm(self.h, _ptr(q), _ptr(k), m, heads, kv_heads, head_dim, pos0, theta,
                                          _ptr(qscale), err, len(err)), err)

    def slerp_residual(self, x, o, lr, rows, width):
        err = _errbuf()
        _check(lib().xtg_hip_slerp_residual(self.h, _ptr(x), _ptr(o), _ptr(lr), rows, width, err, len(err)), err)

    def swiglu_norm(self, g, u, sg, su, rows, width):
        err = _errbuf()
        _check(lib().xtg_hip_swiglu_norm(self.h, _ptr(g), _ptr(u), _ptr(sg), _ptr(su), rows, width, err, len(err)),
               err)

    def gate_norm(self, att, gate, gs, rows, width):
        err = _errbuf()
        _check(lib().xtg_hip_gate_norm(self.h, _ptr(att), _ptr(gate), _ptr(gs), rows, width, err, len(err)), err)

    def add_norm(self, a, b, out, rows, width):
        err = _errbuf()
        _check(lib().xtg_hip_add_norm(self.h, _ptr(a), _ptr(b), _ptr(out), rows, width, err, len(err)), err)

    def read_probe(self, src, nbytes, out):
        """The streaming-read probe: out (device uint32, read_probe_partials(nbytes)) gets the XOR partials of the
        nbytes at src (device)."""
        err = _errbuf()
        _check(lib().xtg_hip_read_probe(self.h, _ptr(src), nbytes, _ptr(out), err, len(err)), err)

    @staticmethod
    def read_probe_partials(nbytes):
        return int(lib().xtg_hip_read_probe_partials(nbytes))

    def argmax(self, logits, rows, n, out):
        """out[r] (device int32) = the first index of the largest of logits[r][:n] (device)."""
        err = _errbuf()
        _check(lib().xtg_hip_argmax(self.h, _ptr(logits), rows, n, _ptr(out), err, len(err)), err)

    def sample(self, logits, rows, n, u, out, temperature=1.0, top_p=1.0, top_k=0, min_p=0.0):
        """out[r] (device int32) = xtg::Sampler::sample of logits[r][:n] (device) with the uniform draw u[r] in
        [0, 1) (host; the reference's generate_canonical draw)."""
        uu = np.ascontiguousarray(u, dtype=np.float64)
        assert uu.shape == (rows,)
        p = Sampling(temperature, top_p, top_k, min_p)
        err = _errbuf()
        _check(lib().xtg_hip_sample(self.h, _ptr(logits), rows, n, ctypes.byref(p), uu.ctypes.data, _ptr(out), err,
                                    len(err)), err)


class DorySession:
    """xtg_hip_dory: forward(x, m, pos0, logits) and prefill(x, n, pos0, want, logits) on device buffers;
    cache(attn, inst) for filling contexts."""

    def __init__(self, backend, weights):
        import xtier_go_amd.workloads as wl
        self.b = backend
        self.w = weights
        cfg, layers, head = wl.dory_structs(weights, Nvfp4, DoryLayer, DoryConfig)
        self._keep = (cfg, layers, head)
        err = _errbuf()
        self.h = lib().xtg_hip_dory_create(backend.h, ctypes.byref(cfg), layers, ctypes.byref(head),
                                           weights.logit_scale.ctypes.data, err, len(err))
        if not self.h:
            raise XtgError(err.value.decode(errors="replace"))
        if getattr(weights, "head_bf16", None) is not None:   # a checkpoint's BF16 LM head
            self.set_head_bf16(weights.head_bf16)

    def destroy(self):
        if self.h:
            lib().xtg_hip_dory_destroy(self.h)
            self.h = None

    def forward(self, x, m, pos0, logits):
        """One chunk of m <= 512 rows; logits for every row."""
        err = _errbuf()
        _check(lib().xtg_hip_dory_forward(self.h, _ptr(x), m, pos0, _ptr(logits), err, len(err)), err)

    def prefill(self, x, n, pos0, want, logits=None):
        """n rows in chunks of up to 512; logits for all rows, the last or none (LOGITS_*)."""
        err = _errbuf()
        _check(lib().xtg_hip_dory_prefill(self.h, _ptr(x), n, pos0, want, _ptr(logits) if logits is not None else None,
                                          err, len(err)), err)

    def set_head_bf16(self, w):
        """A BF16 LM head (uint16 BF16 bits [vocab][hidden], kept referenced) in place of the NVFP4 one."""
        assert w.dtype == np.uint16 and w.flags.c_contiguous
        self._head_bf16 = w
        st = Bf16(w.ctypes.data, w.shape[0], w.shape[1])
        err = _errbuf()
        _check(lib().xtg_hip_dory_head_bf16(self.h, ctypes.byref(st), err, len(err)), err)

    def snapshot(self, slot):
        err = _errbuf()
        _check(lib().xtg_hip_dory_snapshot(self.h, slot, err, len(err)), err)

    def restore(self, slot):
        err = _errbuf()
        _check(lib().xtg_hip_dory_restore(self.h, slot, err, len(err)), err)

    def cache(self, attn, inst=0):
        h = lib().xtg_hip_dory_cache(self.h, attn, inst)
        if not h:
            raise XtgError("no cache %d / %d" % (attn, inst))
        c = KvCache.__new__(KvCache)
        c.b, c.h, c.owned = self.b, h, False
        c.kv_heads, c.head_dim = self.w.cfg["kv_heads"], self.w.cfg["head_dim"]
        return c


class KvCache:
    """A device KV cache (xtg_hip_kv): store from device rows, load to host, save / restore / release."""

    def __init__(self, backend, kv_heads, head_dim, slots, ring=0, dtype=KV_BF16):
        self.b = backend
        self.kv_heads, self.head_dim = kv_heads, head_dim
        self.slots = ring if ring > 0 else slots
        self.ring = ring
        self.owned = True
        err = _errbuf()
        self.h = lib().xtg_hip_kv_create(backend.h, kv_heads, head_dim, slots, ring, dtype, err, len(err))
        if not self.h:
            raise XtgError(err.value.decode(errors="replace"))

    def destroy(self):
        if self.h and self.b.h and self.owned:
            lib().xtg_hip_kv_destroy(self.b.h, self.h)
        self.h = None

    def store(self, pos, n, k, v):
        """Rows pos .. pos + n - 1 from device FP32 k, v [n][kv_heads][head_dim] (queued)."""
        err = _errbuf()
        _check(lib().xtg_hip_kv_store(self.b.h, self.h, pos, n, _ptr(k), _ptr(v), err, len(err)), err)

    def globals(self, k_global, v_global):
        """The two powers of two that an NVFP4 cache's scales are multiplied by; before anything is written."""
        err = _errbuf()
        _check(lib().xtg_hip_kv_globals(self.b.h, self.h, k_global, v_global, err, len(err)), err)

    def write(self, pos, n, k, v, x_dtype=X_F32):
        """store for device rows of x_dtype (queued)."""
        b = self.b
        k, v = _device_rows(b, k, v, n * self.kv_heads * self.head_dim, x_dtype)
        if _lib.xtg_hip_kv_write(b.h, self.h, pos, n, k, v, x_dtype, b._err, _ERR_LEN):
            _check(-1, b._err)

    def read(self, pos, n, k, v, x_dtype=X_F32):
        """The rows of positions pos .. pos + n - 1 as the cache holds them into device k, v [n][kv_heads][head_dim] of
        x_dtype, zeros where it holds none (queued)."""
        b = self.b
        k, v = _device_rows(b, k, v, n * self.kv_heads * self.head_dim, x_dtype)
        if _lib.xtg_hip_kv_read(b.h, self.h, pos, n, k, v, x_dtype, b._err, _ERR_LEN):
            _check(-1, b._err)

    def store_host(self, pos, k, v):
        """Convenience: upload FP32 host rows, then store them."""
        k = np.ascontiguousarray(k, dtype=np.float32)
        v = np.ascontiguousarray(v, dtype=np.float32)
        dk, dv = self.b.array(k), self.b.array(v)
        self.store(pos, k.shape[0], dk, dv)
        self.b.finish()
        dk.free()
        dv.free()

    def load(self, head, p0, p1):
        k = np.empty((p1 - p0, self.head_dim), dtype=np.float32)
        v = np.empty_like(k)
        err = _errbuf()
        _check(lib().xtg_hip_kv_load(self.b.h, self.h, head, p0, p1, k.ctypes.data, v.ctypes.data, err, len(err)), err)
        return k, v

    def nbytes(self):
        return lib().xtg_hip_kv_bytes(self.b.h, self.h)

    def save(self):
        out = np.empty(self.nbytes(), dtype=np.uint8)
        err = _errbuf()
        _check(lib().xtg_hip_kv_save(self.b.h, self.h, out.ctypes.data, out.nbytes, err, len(err)), err)
        return out

    def restore(self, blob):
        blob = np.ascontiguousarray(blob, dtype=np.uint8)
        err = _errbuf()
        _check(lib().xtg_hip_kv_restore(self.b.h, self.h, blob.ctypes.data, blob.nbytes, err, len(err)), err)

    def release(self):
        err = _errbuf()
        _check(lib().xtg_hip_kv_release(self.b.h, self.h, err, len(err)), err)

    def copy_to(self, dst):
        """Device copy of this cache's whole state into dst (same shape, ring and dtype)."""
        err = _errbuf()
        _check(lib().xtg_hip_kv_copy(self.b.h, self.h, dst.h, err, len(err)), err)


class PagedRows:
    """Which sequences the rows of a call belong to, and where their positions lie (HipBackend.paged_rows). The arrays are
    the caller's: what is in them may change between calls, and is read when a call runs."""

    def __init__(self, backend, pos, pages, n_rows=None, starts=None):
        if len(pages.shape) != 2:
            raise XtgError("pages is not [n_seqs][max_pages]")
        if starts is not None and n_rows is None:   # (rows behind one a sequence would be lost)
            raise XtgError("rows with starts want n_rows, the number of the call's rows")
        n_seqs, max_pages = (int(x) for x in pages.shape)
        n_rows = n_seqs if n_rows is None else int(n_rows)
        self.b, self.n_seqs, self.n_rows = backend, n_seqs, n_rows
        self.arrays = pos, pages, starts   # held as long as this is
        self.args = PagedRowsArgs(n_seqs, n_rows, _device_ptr(backend, "pos", pos, n_seqs, _I32),
                                  _device_ptr(backend, "starts", starts, n_seqs + 1, _I32),
                                  _device_ptr(backend, "pages", pages, n_seqs * max_pages, _I32), max_pages)
        self._ref = ctypes.byref(self.args)
        self._own = [a for a in self.arrays if isinstance(a, DeviceArray)]   # whose memory can be freed while they are held

    def of(self, backend):
        """What a call of this backend takes."""
        if backend.device != self.b.device:
            raise XtgError("the rows' positions and pages are not in the memory of the backend's device")
        for a in self._own:
            if not a.ptr or not a.b.h:   # (a backend that is closed frees its arrays)
                raise XtgError("the positions, pages or starts of the rows have been freed")
        return self._ref


class PagedCache:
    """A pool of pages of keys and values (xtg_hip_paged): rows appended, read back, and attended to."""

    def __init__(self, backend, kv_heads, head_dim, pages, page_size=64, dtype=KV_BF16):
        self.b = backend
        self.kv_heads, self.head_dim, self.pages, self.page_size = kv_heads, head_dim, pages, page_size
        err = _errbuf()
        self.h = lib().xtg_hip_paged_create(backend.h, kv_heads, head_dim, pages, page_size, dtype, err, len(err))
        if not self.h:
            raise XtgError(err.value.decode(errors="replace"))

    def destroy(self):
        if self.h and self.b.h:
            lib().xtg_hip_paged_destroy(self.b.h, self.h)
        self.h = None

    def globals(self, k_global, v_global):
        """The two powers of two that an NVFP4 pool's scales are multiplied by; before anything is written."""
        err = _errbuf()
        _check(lib().xtg_hip_paged_globals(self.b.h, self.h, k_global, v_global, err, len(err)), err)

    def append(self, rows, k, v, x_dtype=X_F32, q=None, q_out=None, heads=0, theta=0.0, norm=False, qscale=None,
               q_stride=0, k_stride=0, v_stride=0):
        """Queued: the rows' k and v into their pages, k (and q, into q_out, which may be q) rotated by position (theta 0:
        not) and normalised per head first (norm), q then times qscale (xtg_hip_paged_append). Device rows of x_dtype,
        packed or `stride` elements apart: views of one projection's rows, say."""
        b, kv = self.b, self.kv_heads
        if not k_stride and not v_stride:
            k, v = _device_rows(b, k, v, rows.n_rows * kv * self.head_dim, x_dtype)
        else:
            k = _rows_ptr(b, "k", k, rows.n_rows, kv * self.head_dim, k_stride, x_dtype)
            v = _rows_ptr(b, "v", v, rows.n_rows, kv * self.head_dim, v_stride, x_dtype)
        if q is not None:
            n, width = rows.n_rows, heads * self.head_dim
            if q_stride:
                q, q_out = _rows_ptr(b, "q", q, n, width, q_stride, x_dtype), _rows_ptr(b, "q_out", q_out, n, width, q_stride, x_dtype)
            else:
                q, q_out = _device_ptr(b, "q", q, n * width, x_dtype), _device_ptr(b, "q_out", q_out, n * width, x_dtype)
        if qscale is not None:
            qscale = _device_ptr(b, "qscale", qscale, heads * self.head_dim, X_F32)
        a = PagedAppendArgs(heads, q, q_out, k, v, q_stride, k_stride, v_stride, x_dtype, theta, norm, qscale)
        if _lib.xtg_hip_paged_append(b.h, self.h, rows.of(b), ctypes.byref(a), b._err, _ERR_LEN):
            _check(-1, b._err)

    def read(self, rows, k, v, x_dtype=X_F32):
        """Queued: the rows' k and v as the pages hold them into packed device rows of x_dtype, zeros where there is no
        page (xtg_hip_paged_read)."""
        b = self.b
        k, v = _device_rows(b, k, v, rows.n_rows * self.kv_heads * self.head_dim, x_dtype)
        if _lib.xtg_hip_paged_read(b.h, self.h, rows.of(b), k, v, x_dtype, b._err, _ERR_LEN):
            _check(-1, b._err)

    def attention(self, rows, q, out, heads, x_dtype=X_F32, window=0, scale=None, softcap=0.0, q_stride=0):
        """Queued: attention of the rows over their sequences' pages, their own keys among them (xtg_hip_paged_attention):
        a row at position t sees p <= t, and p > t - window; scores softcap * tanh(scale * q.k / softcap)."""
        b, d = self.b, self.head_dim
        n = rows.n_rows * heads * d
        q = _rows_ptr(b, "q", q, rows.n_rows, heads * d, q_stride, x_dtype) if q_stride else _device_ptr(b, "q", q, n, x_dtype)
        a = PagedAttnArgs(heads, q, q_stride, _device_ptr(b, "out", out, n, x_dtype), x_dtype, window,
                          d ** -0.5 if scale is None else scale, softcap)
        if _lib.xtg_hip_paged_attention(b.h, self.h, rows.of(b), ctypes.byref(a), b._err, _ERR_LEN):
            _check(-1, b._err)


class DeviceArray:
    """Device memory from xtg_hip_alloc with a numpy shape and dtype (the library's own buffers, so no other
    HIP runtime is involved)."""

    def __init__(self, backend, a=None, shape=None, dtype=np.float32):
        self.b = backend
        if a is not None:
            a = np.ascontiguousarray(a)
            shape, dtype = a.shape, a.dtype
        self.shape = tuple(shape)
        self.dtype = np.dtype(dtype)
        self.nbytes = int(np.prod(self.shape)) * self.dtype.itemsize
        self.ptr = backend.alloc(max(self.nbytes, 4))
        if a is not None:
            backend.write(self.ptr, a)

    def data_ptr(self):
        return self.ptr

    def upload(self, a):
        a = np.ascontiguousarray(a, dtype=self.dtype)
        assert a.nbytes == self.nbytes
        self.b.write(self.ptr, a)

    def numpy(self):
        out = np.empty(self.shape, dtype=self.dtype)
        return self.b.read(self.ptr, out)

    def free(self):
        if self.ptr:
            self.b.release(self.ptr)
            self.ptr = None
