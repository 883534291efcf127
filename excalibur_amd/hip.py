"""ctypes binding of the exhip C ABI (include/exhip.h) with numpy at the host boundary.

This is the Python face of the product library: it loads excalibur_amd/lib/libexhip.so and fails
loudly if that library or a gfx950 device is missing. There is no CPU fallback.
"""
import ctypes
import functools
import math
import os

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libexhip.so")

I8, F16, F32 = 0, 1, 2
_NP = {I8: np.int8, F16: np.uint16, F32: np.float32}


class ExhipError(RuntimeError):
    pass


class ConvDesc(ctypes.Structure):
    _fields_ = [(k, ctypes.c_int) for k in
                ("n", "c", "h", "w", "k", "kh", "kw", "sh", "sw", "pt", "pb", "pl", "pr", "act", "c_stride", "k_stride",
                 "post_relu")] + [("fs_out", ctypes.c_float), ("post_op", ctypes.c_int), ("post_alpha", ctypes.c_float),
                                  ("post_beta", ctypes.c_float), ("post_slope", ctypes.c_void_p),
                                  ("post_slope_shared", ctypes.c_int), ("residual_last", ctypes.c_int),
                                  ("post_bn_a", ctypes.c_void_p), ("post_bn_b", ctypes.c_void_p), ("exact_k", ctypes.c_int)]


_lib = None


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ExhipError(f"{LIB_PATH} is not built; run `python -c 'import __graft_entry__ as g; g.build()'` "
                             "or `make -C excalibur_amd/csrc`")
        L = ctypes.CDLL(LIB_PATH)
        L.exhip_last_error.restype = ctypes.c_char_p
        L.exhip_conv_packed_bytes.restype = ctypes.c_size_t
        L.exhip_static_scratch_bytes.restype = ctypes.c_size_t
        L.exhip_host_alloc.restype = ctypes.c_void_p
        L.exhip_host_alloc.argtypes = [ctypes.c_size_t]
        L.exhip_host_free.restype = None
        L.exhip_host_free.argtypes = [ctypes.c_void_p]
        L.exhip_f8_packed_bytes.restype = ctypes.c_size_t
        L.exhip_i8_packed_bytes.restype = ctypes.c_size_t
        L.exhip_log_probabilities_workspace.restype = ctypes.c_size_t
        _lib = L
    return _lib


def set_option(name, value):
    """Test / development switches of the library (exhip_set_option)."""
    _check(lib().exhip_set_option(name.encode(), int(value)))


ERR_UNSUPPORTED = 10002  # a form that an entry point leaves to others


def _check(rc):
    if rc != 0:
        raise ExhipError(f"exhip error {rc}: {lib().exhip_last_error().decode()}")


def pad_to(v, m):
    return (v + m - 1) // m * m


class DevArray:
    """A device allocation with a logical numpy shape/dtype."""

    def __init__(self, ctx, shape, dtype):
        self.ctx = ctx
        self.shape = tuple(int(s) for s in shape)
        self.dtype = np.dtype(dtype)
        self.char = self.dtype.char if self.dtype.isnative else self.dtype.str
        self.size = math.prod(self.shape)
        self.nbytes = self.size * self.dtype.itemsize
        p = ctypes.c_void_p()
        _check(lib().exhip_malloc(ctx.h, ctypes.c_size_t(self.nbytes), ctypes.byref(p)))
        self.ptr = p

    def upload(self, a):
        a = np.ascontiguousarray(a, self.dtype)
        assert a.nbytes == self.nbytes, (a.shape, self.shape)
        _check(lib().exhip_memcpy_h2d(self.ctx.h, self.ptr, a.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(self.nbytes)))
        return self

    def download(self):
        out = np.empty(self.shape, self.dtype)
        _check(lib().exhip_memcpy_d2h(self.ctx.h, out.ctypes.data_as(ctypes.c_void_p), self.ptr, ctypes.c_size_t(self.nbytes)))
        return out

    def zero(self):
        _check(lib().exhip_memset(self.ctx.h, self.ptr, 0, ctypes.c_size_t(self.nbytes)))
        return self

    def free(self):
        if self.ptr:
            _check(lib().exhip_free(self.ctx.h, self.ptr))
            self.ptr = None

    def at(self, offset_bytes):
        """Something with a .ptr that many bytes into the allocation (an operand that starts inside a larger tensor)."""
        assert 0 <= offset_bytes < self.nbytes
        return _Inside(ctypes.c_void_p(self.ptr.value + int(offset_bytes)))


class _Inside:
    char, size = "", math.inf

    def __init__(self, ptr):
        self.ptr = ptr


class View:
    """Device memory that something else owns (another library's tensor), with a shape and dtype: what the calls below need of an operand. It has to
    outlive the work queued on it."""

    def __init__(self, address, shape, dtype):
        self.ptr = ctypes.c_void_p(int(address))
        self.shape = tuple(int(s) for s in shape)
        self.dtype = np.dtype(dtype)
        self.char = self.dtype.char if self.dtype.isnative else self.dtype.str
        self.size = math.prod(self.shape)


class F8Desc(ctypes.Structure):
    _fields_ = [(k, ctypes.c_int) for k in ("m", "n_out", "k_in", "x_stride", "y_stride")]
    _counts = None

    def __setattr__(self, name, value):
        super().__setattr__(name, value)
        if name != "_counts":
            self._counts = None

    def counts(self):
        """How many values the products' operands have: rows, their scales, packed bytes of one projection, its scales, a bias, a result, a quantized one's
        scales. Counted once: a call that checks its operands is made for every row of a serving program."""
        m, n, k = self.m, self.n_out, self.k_in
        bn, bk = _blocks(n), _blocks(k)
        self._counts = (m - 1) * self.x_stride + k, bk * m, -(-n // 16) * bk * 2048, bn * bk, n, (m - 1) * self.y_stride + n, bn * m
        return self._counts


class I8Desc(ctypes.Structure):
    _fields_ = [(k, ctypes.c_int) for k in ("m", "n_out", "k_in", "x_stride", "y_stride")]
    _counts = None

    def __setattr__(self, name, value):
        super().__setattr__(name, value)
        if name != "_counts":
            self._counts = None

    def counts(self, experts=1, gated=False):
        """Of how many experts and which product this is, and how many values its operands have: rows of the input where there are as many as of the result, packed
        bytes, scales of the outputs, a result. Counted once for the calls that follow."""
        packed = Ctx.i8_packed_bytes(self.n_out, self.k_in, gated, experts)
        self._counts = (experts, gated), (self.m - 1) * self.x_stride + self.k_in, packed, experts * self.n_out, (self.m - 1) * self.y_stride + self.n_out
        return self._counts


F8_BLOCK = 128  # values that share a scale


class Event:
    def __init__(self):
        self.h = ctypes.c_void_p()
        _check(lib().exhip_event_create(ctypes.byref(self.h)))

    def record(self, ctx):
        _check(lib().exhip_event_record(ctx.h, self.h))

    def destroy(self):
        if self.h:
            _check(lib().exhip_event_destroy(self.h))
            self.h = None

    def elapsed_ms(self, stop):
        ms = ctypes.c_float()
        _check(lib().exhip_event_elapsed_ms(self.h, stop.h, ctypes.byref(ms)))
        return ms.value


def _ptr(a):
    return a.ptr if a is not None else None


_FLOATS, _HALVES, _ROWS, _CODES, _IDS = "f", "He", "fHe", "Bb", "i"  # numpy's characters of the types that an operand may have


def _refused(*operands):
    """Says which operand (its name, itself, the values that the call reads or writes, its types) is of another type or too small."""
    for name, a, count, types in operands:
        if a is not None and a.char not in types:
            raise ExhipError(f"{name} is {a.dtype}, not {' or '.join(np.dtype(t).name for t in types)}")
        if a is not None and a.size < count:
            raise ExhipError(f"{name} has {a.size} values, the call takes {count}")


def _holds(a, count, types):
    """Whether an operand that is there has values of one of the types, and enough. (An address alone, DevArray.at(), says neither.)"""
    return a is None or (a.size >= count and a.char in types)


_MOST = 2 ** 31 - 1  # of a C int; ctypes would cut larger ones


def _size_refused(*sizes):
    raise ExhipError(f"{sizes}: more than a size of the library holds")


def _blocks(v):
    return -(-v // F8_BLOCK)


class Ctx:
    def __init__(self, device=0):
        self.h = ctypes.c_void_p()
        _check(lib().exhip_init(int(device), ctypes.byref(self.h)))

    def close(self):
        if self.h:
            lib().exhip_destroy(self.h)
            self.h = None

    def device_name(self):
        buf = ctypes.create_string_buffer(256)
        _check(lib().exhip_device_name(self.h, buf, ctypes.c_size_t(256)))
        return buf.value.decode()

    def sync(self):
        _check(lib().exhip_sync(self.h))

    def empty(self, shape, dtype):
        return DevArray(self, shape, dtype)

    def array(self, a, dtype=None):
        a = np.ascontiguousarray(a, dtype if dtype is not None else a.dtype)
        return DevArray(self, a.shape, a.dtype).upload(a)

    @staticmethod
    def view(address, shape, dtype):
        """An operand at a device address that the caller owns."""
        return View(address, shape, dtype)

    # ---- layout / precision ----
    def quantize_nchw_to_nhwc_i8(self, x, fs, c_stride, fs_per_channel=None):
        n, c, h, w = x.shape
        y = self.empty((n, h, w, c_stride), np.int8)
        _check(lib().exhip_quantize_nchw_f32_to_nhwc_i8(self.h, x.ptr, n, c, h, w, ctypes.c_float(float(fs)),
                                                       _ptr(fs_per_channel), c_stride, y.ptr))
        return y

    def nchw_to_nhwc(self, x, c_stride, out="f32"):
        n, c, h, w = x.shape
        if x.dtype == np.float32 and out == "f32":
            y = self.empty((n, h, w, c_stride), np.float32)
            _check(lib().exhip_nchw_f32_to_nhwc_f32(self.h, x.ptr, n, c, h, w, c_stride, y.ptr))
        elif x.dtype == np.float32 and out == "f16":
            y = self.empty((n, h, w, c_stride), np.uint16)
            _check(lib().exhip_nchw_f32_to_nhwc_f16(self.h, x.ptr, n, c, h, w, c_stride, y.ptr))
        else:
            y = self.empty((n, h, w, c_stride), np.uint16)
            _check(lib().exhip_nchw_f16_to_nhwc_f16(self.h, x.ptr, n, c, h, w, c_stride, y.ptr))
        return y

    def nhwc_to_nchw(self, x, c, out="f32"):
        n, h, w, cs = x.shape
        if x.dtype == np.float32:
            y = self.empty((n, c, h, w), np.float32)
            _check(lib().exhip_nhwc_f32_to_nchw_f32(self.h, x.ptr, n, c, h, w, cs, y.ptr))
        elif out == "f32":
            y = self.empty((n, c, h, w), np.float32)
            _check(lib().exhip_nhwc_f16_to_nchw_f32(self.h, x.ptr, n, c, h, w, cs, y.ptr))
        else:
            y = self.empty((n, c, h, w), np.uint16)
            _check(lib().exhip_nhwc_f16_to_nchw_f16(self.h, x.ptr, n, c, h, w, cs, y.ptr))
        return y

    def f32_to_f16(self, x):
        y = self.empty(x.shape, np.uint16)
        _check(lib().exhip_f32_to_f16(self.h, x.ptr, y.ptr, ctypes.c_size_t(x.size)))
        return y

    def f16_to_f32(self, x):
        y = self.empty(x.shape, np.float32)
        _check(lib().exhip_f16_to_f32(self.h, x.ptr, y.ptr, ctypes.c_size_t(x.size)))
        return y

    # ---- convolution ----
    @staticmethod
    def conv_desc(n, c, h, w, k, kernel, stride=1, pad=0, act=0, c_stride=None, k_stride=None, post_relu=0, fs_out=0.0,
                  post_op=None, post_alpha=0.0, post_beta=0.0, residual_last=0, post_bn=None, exact_k=0):
        kh, kw = (kernel, kernel) if np.isscalar(kernel) else kernel
        sh, sw = (stride, stride) if np.isscalar(stride) else stride
        pt, pb, pl, pr = (pad,) * 4 if np.isscalar(pad) else pad
        return ConvDesc(n, c, h, w, k, kh, kw, sh, sw, pt, pb, pl, pr, act, c_stride if c_stride else c,
                        k_stride if k_stride else k, post_relu, fs_out, 0 if post_op is None else 1 + Ctx.UNARY[post_op],
                        post_alpha, post_beta, None, 0, residual_last, post_bn[0].ptr if post_bn else None,
                        post_bn[1].ptr if post_bn else None, int(exact_k))

    @staticmethod
    def conv_out_hw(d):
        oh, ow = ctypes.c_int(), ctypes.c_int()
        _check(lib().exhip_conv_out_hw(ctypes.byref(d), ctypes.byref(oh), ctypes.byref(ow)))
        return oh.value, ow.value

    def pack_conv_weights(self, d, dtype, w_oihw):
        nbytes = lib().exhip_conv_packed_bytes(ctypes.byref(d), dtype)
        if nbytes == 0:
            raise ExhipError(f"exhip_conv_packed_bytes: {lib().exhip_last_error().decode()}")
        w = np.ascontiguousarray(w_oihw, _NP[dtype])
        packed = np.empty(nbytes, np.uint8)
        _check(lib().exhip_conv_pack_weights(ctypes.byref(d), dtype, w.ctypes.data_as(ctypes.c_void_p),
                                             packed.ctypes.data_as(ctypes.c_void_p)))
        return self.array(packed)

    def conv2d_i8(self, d, x, wp, scale, bias=None, residual=None, y_i8=None, y_f32_nhwc=None, y_f32_nchw=None, acc=None):
        _check(lib().exhip_conv2d_i8(self.h, ctypes.byref(d), x.ptr, wp.ptr, scale.ptr, _ptr(bias), _ptr(residual),
                                     _ptr(y_i8), _ptr(y_f32_nhwc), _ptr(y_f32_nchw), _ptr(acc)))

    def conv2d_i8_maxpool3x3s2(self, d, pool_pad, pool_oh, pool_ow, x, wp, scale, bias=None, y_i8=None, y_f32_nhwc=None):
        _check(lib().exhip_conv2d_i8_maxpool3x3s2(self.h, ctypes.byref(d), pool_pad, pool_pad, pool_oh, pool_ow, x.ptr, wp.ptr,
                                                  scale.ptr, _ptr(bias), _ptr(y_i8), _ptr(y_f32_nhwc)))

    def stem_f32_conv_i8_maxpool3x3s2(self, d, pool_pad, pool_oh, pool_ow, x_nchw, fs_in, wp, scale, scales_nonnegative, bias=None,
                                      y_i8=None, y_f32_nhwc=None):
        """Returns False when the library leaves the shape to the quantizer + exhip_conv2d_i8_maxpool3x3s2."""
        rc = lib().exhip_stem_f32_conv_i8_maxpool3x3s2(self.h, ctypes.byref(d), pool_pad, pool_pad, pool_oh, pool_ow, x_nchw.ptr,
                                                       ctypes.c_float(fs_in), wp.ptr, scale.ptr, int(scales_nonnegative), _ptr(bias),
                                                       _ptr(y_i8), _ptr(y_f32_nhwc))
        if rc == 10002:
            return False
        _check(rc)
        return True

    def conv2d_i8_projection(self, d, x, wp, scale, bias, d_proj, x_proj, wp_proj, scale_proj, bias_proj, y_i8, y_f32_nhwc):
        """Returns False when the library leaves the pair to two exhip_conv2d_i8 calls."""
        rc = lib().exhip_conv2d_i8_projection(self.h, ctypes.byref(d), x.ptr, wp.ptr, scale.ptr, _ptr(bias), ctypes.byref(d_proj),
                                              x_proj.ptr, wp_proj.ptr, scale_proj.ptr, _ptr(bias_proj), y_i8.ptr, y_f32_nhwc.ptr)
        if rc == 10002:
            return False
        _check(rc)
        return True

    def conv2d_f16(self, d, x, wp, bias=None, residual=None, y_f16_nhwc=None, y_f16_nchw=None, y_f32_nchw=None):
        _check(lib().exhip_conv2d_f16(self.h, ctypes.byref(d), x.ptr, wp.ptr, _ptr(bias), _ptr(residual), _ptr(y_f16_nhwc),
                                      _ptr(y_f16_nchw), _ptr(y_f32_nchw)))

    def conv2d_grouped(self, d, group, x, wp, bias, y, scale=None):
        """A detection head (y: n x k / group x pixels x group): int8 with `scale`, else fp16."""
        if scale is not None:
            _check(lib().exhip_conv2d_i8_grouped(self.h, ctypes.byref(d), group, x.ptr, wp.ptr, scale.ptr, _ptr(bias), y.ptr))
        else:
            _check(lib().exhip_conv2d_f16_grouped(self.h, ctypes.byref(d), group, x.ptr, wp.ptr, _ptr(bias), y.ptr))

    def conv2d_f32(self, d, x, wp, bias=None, residual=None, y_f32_nhwc=None, y_f32_nchw=None):
        _check(lib().exhip_conv2d_f32(self.h, ctypes.byref(d), x.ptr, wp.ptr, _ptr(bias), _ptr(residual), _ptr(y_f32_nhwc),
                                      _ptr(y_f32_nchw)))

    def conv2d_direct(self, d, groups, x, y, w_f32=None, w_i8=None, fs=1.0, scale=None, bias=None):
        _check(lib().exhip_conv2d_direct_nchw(self.h, ctypes.byref(d), groups, x.ptr, _ptr(w_f32), _ptr(w_i8),
                                              ctypes.c_float(float(fs)), _ptr(scale), _ptr(bias), y.ptr))

    # ---- bandwidth-bound operators ----
    def dwconv3x3_nchw_f32(self, x, w9, bias, stride, pad, act):
        n, c, h, w = x.shape
        pt, pb, pl, pr = (pad,) * 4 if np.isscalar(pad) else pad
        oh, ow = (h + pt + pb - 3) // stride + 1, (w + pl + pr - 3) // stride + 1
        y = self.empty((n, c, oh, ow), np.float32)
        _check(lib().exhip_dwconv3x3_nchw_f32(self.h, x.ptr, w9.ptr, _ptr(bias), y.ptr, n, c, h, w, stride, pt, pb, pl, pr, act))
        return y

    def dwconv3x3_nhwc_f16(self, x, c, w9, bias, stride, pad, act):
        n, h, w, cs = x.shape
        pt, pb, pl, pr = (pad,) * 4 if np.isscalar(pad) else pad
        oh, ow = (h + pt + pb - 3) // stride + 1, (w + pl + pr - 3) // stride + 1
        y = self.empty((n, oh, ow, cs), np.uint16)
        _check(lib().exhip_dwconv3x3_nhwc_f16(self.h, x.ptr, w9.ptr, _ptr(bias), y.ptr, n, c, h, w, cs, stride, pt, pb, pl, pr,
                                              act))
        return y

    def dwconv3x3_nchw_f32_prelu(self, x, w9, bias, slope, shared, stride, pad):
        n, c, h, w = x.shape
        pt, pb, pl, pr = (pad,) * 4 if np.isscalar(pad) else pad
        oh, ow = (h + pt + pb - 3) // stride + 1, (w + pl + pr - 3) // stride + 1
        y = self.empty((n, c, oh, ow), np.float32)
        _check(lib().exhip_dwconv3x3_nchw_f32_prelu(self.h, x.ptr, w9.ptr, _ptr(bias), slope.ptr, int(shared), y.ptr, n, c, h, w,
                                                    stride, pt, pb, pl, pr))
        return y

    def dwconv3x3_nhwc_f16_prelu(self, x, c, w9, bias, slope, shared, stride, pad):
        n, h, w, cs = x.shape
        pt, pb, pl, pr = (pad,) * 4 if np.isscalar(pad) else pad
        oh, ow = (h + pt + pb - 3) // stride + 1, (w + pl + pr - 3) // stride + 1
        y = self.empty((n, oh, ow, cs), np.uint16)
        _check(lib().exhip_dwconv3x3_nhwc_f16_prelu(self.h, x.ptr, w9.ptr, _ptr(bias), slope.ptr, int(shared), y.ptr, n, c, h, w,
                                                    cs, stride, pt, pb, pl, pr))
        return y

    def dw_dequant_weights(self, w_i8, ws):
        k = w_i8.shape[0]
        wf = self.empty(w_i8.shape, np.float32)
        _check(lib().exhip_dw_dequant_weights(self.h, w_i8.ptr, ws.ptr, wf.ptr, k, w_i8.size // k))
        return wf

    @staticmethod
    def pool_out_hw(h, w, kh, kw, sh, sw, pt, pb, pl, pr, pad_mode):
        oh, ow = ctypes.c_int(), ctypes.c_int()
        _check(lib().exhip_pool_out_hw(h, w, kh, kw, sh, sw, pt, pb, pl, pr, pad_mode, ctypes.byref(oh), ctypes.byref(ow)))
        return oh.value, ow.value

    @staticmethod
    def _pool_args(h, w, kernel, stride, pad, global_pool, pad_mode):
        kh, kw = (kernel, kernel) if np.isscalar(kernel) else kernel
        sh, sw = (stride, stride) if np.isscalar(stride) else stride
        pt, pb, pl, pr = (pad,) * 4 if np.isscalar(pad) else pad
        if global_pool:  # src/Excalibur/operation_pooling.cpp:90-100
            kh, kw, sh, sw, pt, pb, pl, pr = h, w, 1, 1, 0, 0, 0, 0
        oh, ow = Ctx.pool_out_hw(h, w, kh, kw, sh, sw, pt, pb, pl, pr, pad_mode)
        return kh, kw, sh, sw, pt, pb, pl, pr, oh, ow

    def pool2d_nchw_f32(self, x, ptype, kernel=0, stride=1, pad=0, global_pool=False, pad_mode=1, count_include_pad=0):
        n, c, h, w = x.shape
        kh, kw, sh, sw, pt, pb, pl, pr, oh, ow = self._pool_args(h, w, kernel, stride, pad, global_pool, pad_mode)
        y = self.empty((n, c, oh, ow), np.float32)
        _check(lib().exhip_pool2d_nchw_f32(self.h, x.ptr, y.ptr, n, c, h, w, oh, ow, ptype, kh, kw, sh, sw, pt, pb, pl, pr,
                                           count_include_pad))
        return y

    def maxpool2d_nhwc_f32(self, x, c, kernel, stride, pad, fs_out=None, want_f32=True):
        n, h, w, cs = x.shape
        kh, kw, sh, sw, pt, pb, pl, pr, oh, ow = self._pool_args(h, w, kernel, stride, pad, False, 1)
        y = self.empty((n, oh, ow, cs), np.float32) if want_f32 else None
        yq = self.empty((n, oh, ow, cs), np.int8) if fs_out is not None else None
        _check(lib().exhip_maxpool2d_nhwc_f32(self.h, x.ptr, _ptr(y), _ptr(yq), ctypes.c_float(float(fs_out or 0.0)), n, c, h,
                                              w, cs, oh, ow, kh, kw, sh, sw, pt, pl))
        return y, yq

    def pool2d_nhwc_f16(self, x, c, ptype, kernel=0, stride=1, pad=0, global_pool=False, pad_mode=1, count_include_pad=0):
        n, h, w, cs = x.shape
        kh, kw, sh, sw, pt, pb, pl, pr, oh, ow = self._pool_args(h, w, kernel, stride, pad, global_pool, pad_mode)
        y = self.empty((n, oh, ow, cs), np.uint16)
        _check(lib().exhip_pool2d_nhwc_f16(self.h, x.ptr, y.ptr, n, c, h, w, cs, oh, ow, ptype, kh, kw, sh, sw, pt, pb, pl, pr,
                                           count_include_pad))
        return y

    def maxpool_same_nhwc_f16(self, x, k, y=None, tmp=None):
        """Stride-1 max pooling with window k and padding k // 2 on an NHWC half tensor; tmp is the caller's workspace."""
        n, h, w, c = x.shape
        y = y if y is not None else self.empty(x.shape, np.uint16)
        tmp = tmp if tmp is not None else self.empty(x.shape, np.uint16)
        _check(lib().exhip_maxpool_same_nhwc_f16(self.h, x.ptr, tmp.ptr, y.ptr, n, c, h, w, int(k)))
        return y

    def maxpool_same_nhwc_f16_static(self, x, k, y):
        """The same through the entry point that allocates nothing: y is preallocated by the caller."""
        n, h, w, c = x.shape
        _check(lib().exhip_maxpool_same_nhwc_f16_static(self.h, x.ptr, y.ptr, n, c, h, w, int(k)))
        return y

    def eltwise_f32(self, inputs, etype, coeffs=None):
        ptrs = (ctypes.c_void_p * len(inputs))(*[a.ptr.value for a in inputs])
        co = None
        if coeffs is not None:
            co = (ctypes.c_float * len(inputs))(*[float(v) for v in coeffs])
        y = self.empty(inputs[0].shape, np.float32)
        _check(lib().exhip_eltwise_f32(self.h, ptrs, len(inputs), co, etype, y.ptr, ctypes.c_size_t(y.size)))
        return y

    def add_f32(self, a, b, relu=False):
        y = self.empty(a.shape, np.float32)
        _check(lib().exhip_add_f32(self.h, a.ptr, b.ptr, y.ptr, ctypes.c_size_t(y.size), int(relu)))
        return y

    def relu_f32(self, x):
        y = self.empty(x.shape, np.float32)
        _check(lib().exhip_relu_f32(self.h, x.ptr, y.ptr, ctypes.c_size_t(y.size)))
        return y

    # ---- activation / glue layers ----
    UNARY = {"hardswish": 0, "leakyrelu": 1, "sigmoid": 2, "hardsigmoid": 3, "clip": 4}
    CHANNEL = {"prelu": 0, "batchnorm": 1, "input": 2}

    def unary_f32(self, op, x, alpha=0.0, beta=0.0):
        y = self.empty(x.shape, np.float32)
        _check(lib().exhip_unary_f32(self.h, self.UNARY[op], x.ptr, y.ptr, ctypes.c_size_t(y.size), ctypes.c_float(float(alpha)),
                                     ctypes.c_float(float(beta))))
        return y

    def channelwise_f32(self, op, x, p0, p1=None, shared=False):
        n, c, h, w = x.shape
        y = self.empty(x.shape, np.float32)
        _check(lib().exhip_channelwise_f32(self.h, self.CHANNEL[op], x.ptr, y.ptr, n, c, h * w, p0.ptr, _ptr(p1), int(shared)))
        return y

    def unary_f16(self, op, x, alpha=0.0, beta=0.0):
        y = self.empty(x.shape, np.uint16)
        _check(lib().exhip_unary_f16(self.h, self.UNARY[op], x.ptr, y.ptr, ctypes.c_size_t(y.size), ctypes.c_float(float(alpha)),
                                     ctypes.c_float(float(beta))))
        return y

    def channelwise_f16(self, op, x, p0, p1=None, shared=False):
        n, c, h, w = x.shape
        y = self.empty(x.shape, np.uint16)
        _check(lib().exhip_channelwise_f16(self.h, self.CHANNEL[op], x.ptr, y.ptr, n, c, h * w, p0.ptr, _ptr(p1), int(shared)))
        return y

    def channelwise_nhwc_f16(self, op, x, p0, p1=None, shared=False):
        n, h, w, c = x.shape
        y = self.empty(x.shape, np.uint16)
        _check(lib().exhip_channelwise_nhwc_f16(self.h, self.CHANNEL[op], x.ptr, y.ptr, ctypes.c_size_t(n * h * w), c, p0.ptr, _ptr(p1),
                                                int(shared)))
        return y

    def concat_nhwc_f32(self, inputs, channels, out_stride, bn=None, unary=None, alpha=0.0, beta=0.0, want_f32=True, fs_out=None):
        """Channel blocks of float32 NHWC blobs (inputs[i] has channels[i] channels at a stride of its last dimension) side by
        side, BatchNorm bn=(a, b) and the activation `unary` behind them, as float32 NHWC and / or int8 NHWC q8(v * fs_out)
        (exhip_concat_batchnorm_unary_nhwc_f32). Returns (float32 or None, int8 or None)."""
        n, h, w, _ = inputs[0].shape
        ptrs = (ctypes.c_void_p * len(inputs))(*[a.ptr.value for a in inputs])
        ch = (ctypes.c_int * len(inputs))(*channels)
        st = (ctypes.c_int * len(inputs))(*[a.shape[3] for a in inputs])
        y_f = self.empty((n, h, w, out_stride), np.float32) if want_f32 else None
        y_q = self.empty((n, h, w, out_stride), np.int8) if fs_out is not None else None
        _check(lib().exhip_concat_batchnorm_unary_nhwc_f32(self.h, ptrs, ch, st, len(inputs), ctypes.c_size_t(n * h * w),
                                                           _ptr(bn[0] if bn else None), _ptr(bn[1] if bn else None),
                                                           -1 if unary is None else self.UNARY[unary], ctypes.c_float(float(alpha)),
                                                           ctypes.c_float(float(beta)), int(out_stride), _ptr(y_f), _ptr(y_q),
                                                           ctypes.c_float(float(fs_out or 0.0))))
        return y_f, y_q

    def concat_nhwc_f16(self, inputs, bn=None, unary=None, alpha=0.0, beta=0.0):
        """Concat of NHWC half blobs along the channels; with bn=(a, b) and / or unary= the BatchNorm and activation layers
        behind it in the same kernel (exhip_concat_batchnorm_unary_nhwc_f16), else the plain exhip_concat_channels_nhwc_f16."""
        n, h, w, _ = inputs[0].shape
        ptrs = (ctypes.c_void_p * len(inputs))(*[a.ptr.value for a in inputs])
        ch = (ctypes.c_int * len(inputs))(*[a.shape[3] for a in inputs])
        y = self.empty((n, h, w, sum(a.shape[3] for a in inputs)), np.uint16)
        if bn is None and unary is None:
            _check(lib().exhip_concat_channels_nhwc_f16(self.h, ptrs, ch, len(inputs), ctypes.c_size_t(n * h * w), y.ptr))
        else:
            _check(lib().exhip_concat_batchnorm_unary_nhwc_f16(self.h, ptrs, ch, len(inputs), ctypes.c_size_t(n * h * w),
                                                               _ptr(bn[0] if bn else None), _ptr(bn[1] if bn else None),
                                                               -1 if unary is None else self.UNARY[unary], ctypes.c_float(float(alpha)),
                                                               ctypes.c_float(float(beta)), y.ptr))
        return y

    def concat_channels_f32(self, inputs):
        n, _, h, w = inputs[0].shape
        ptrs = (ctypes.c_void_p * len(inputs))(*[a.ptr.value for a in inputs])
        ch = (ctypes.c_int * len(inputs))(*[a.shape[1] for a in inputs])
        y = self.empty((n, sum(a.shape[1] for a in inputs), h, w), np.float32)
        _check(lib().exhip_concat_channels_f32(self.h, ptrs, ch, len(inputs), n, h * w, y.ptr))
        return y

    def interp_nearest_f32(self, x, oh, ow):
        n, c, h, w = x.shape
        y = self.empty((n, c, oh, ow), np.float32)
        _check(lib().exhip_interp_nearest_f32(self.h, x.ptr, y.ptr, n, c, h, w, oh, ow))
        return y

    def focus_f32(self, x):
        n, c, h, w = x.shape
        y = self.empty((n, 4 * c, h // 2, w // 2), np.float32)
        _check(lib().exhip_focus_f32(self.h, x.ptr, y.ptr, n, c, h, w))
        return y

    def focus_f16(self, x):
        n, c, h, w = x.shape
        y = self.empty((n, 4 * c, h // 2, w // 2), np.uint16)
        _check(lib().exhip_focus_f16(self.h, x.ptr, y.ptr, n, c, h, w))
        return y

    def maxpool2d_nhwc_i8(self, x, c, kernel, stride, pad, oh, ow):
        """MAX pooling on an int8 NHWC tensor [n, h, w, c_stride] (exhip_maxpool2d_nhwc_i8); pad = (top, left)."""
        n, h, w, cs = x.shape
        y = self.empty((n, oh, ow, cs), np.int8)
        _check(lib().exhip_maxpool2d_nhwc_i8(self.h, x.ptr, y.ptr, n, int(c), h, w, cs, int(oh), int(ow), int(kernel), int(kernel), int(stride),
                                             int(stride), int(pad[0]), int(pad[1])))
        return y


    def maxpool_same_pyramid_nhwc_i8(self, x, c, k, levels=3):
        """Stride-1 "same" max pools of window k applied `levels` times to an int8 NHWC tensor, every level's result returned
        (exhip_maxpool_same_pyramid_nhwc_i8)."""
        n, h, w, cs = x.shape
        ys = [self.empty((n, h, w, cs), np.int8) for _ in range(levels)]
        ptrs = [y.ptr for y in ys] + [None] * (3 - levels)
        _check(lib().exhip_maxpool_same_pyramid_nhwc_i8(self.h, x.ptr, ptrs[0], ptrs[1], ptrs[2], n, int(c), h, w, cs, int(k)))
        return ys
    def input_focus_quantize(self, x, means, scales, fs, c_stride=32):
        """Input layer, YoloV5Focus and the int8 quantizer in one pass (exhip_input_focus_quantize_nchw_f32_to_nhwc_i8): float32
        NCHW -> int8 NHWC [n, h / 2, w / 2, c_stride]. Returns None where the library leaves the shape to the three layers."""
        n, c, h, w = x.shape
        y = self.empty((n, h // 2, w // 2, c_stride), np.int8)
        m = (ctypes.c_float * len(means))(*[float(v) for v in means])
        sc = (ctypes.c_float * len(scales))(*[float(v) for v in scales])
        rc = lib().exhip_input_focus_quantize_nchw_f32_to_nhwc_i8(self.h, x.ptr, n, c, h, w, m, sc, ctypes.c_float(float(fs)), int(c_stride), y.ptr)
        if rc == 10002:
            return None
        _check(rc)
        return y

    def nhwc_to_grouped_f32(self, x, channels, groups):
        """[n, h, w, stride] float32 with `channels` = groups * per_group real channels -> [n, groups, h * w, per_group]
        (exhip_nhwc_f32_to_grouped_f32): a detection head's Reshape + Transpose on the NHWC result."""
        n, h, w, stride = x.shape
        per_group = channels // groups
        y = self.empty((n, groups, h * w, per_group), np.float32)
        _check(lib().exhip_nhwc_f32_to_grouped_f32(self.h, x.ptr, n, h * w, int(groups), int(per_group), int(stride), y.ptr))
        return y

    def binaryop_f32(self, op, mode, large, small):
        """op 0 ADD / 1 SUB / 2 MUL / 3 DIV; mode 0 equal shapes, 1 per image, 2 per (image, channel), 3 per (image, pixel)."""
        n, c, h, w = large.shape
        y = self.empty(large.shape, np.float32)
        _check(lib().exhip_binaryop_f32(self.h, int(op), int(mode), large.ptr, small.ptr, y.ptr, n, c, h * w, small.shape[0]))
        return y

    def softmax_channels_f32(self, x):
        n, c = x.shape[:2]
        y = self.empty(x.shape, np.float32)
        _check(lib().exhip_softmax_channels_f32(self.h, x.ptr, y.ptr, n, c, int(np.prod(x.shape[2:], dtype=np.int64))))
        return y

    def transpose_hw_f32(self, x):
        n, c, h, w = x.shape
        y = self.empty((n, c, w, h), np.float32)
        _check(lib().exhip_transpose_hw_f32(self.h, x.ptr, y.ptr, n * c, h, w))
        return y

    def transpose_hw_f16(self, x):
        n, c, h, w = x.shape
        y = self.empty((n, c, w, h), np.uint16)
        _check(lib().exhip_transpose_hw_f16(self.h, x.ptr, y.ptr, n * c, h, w))
        return y

    def deconv2d_f32(self, x, w, bias, stride, pad):
        n, c, h, wd = x.shape
        _, k, kh, kw = w.shape
        sh, sw = (stride, stride) if np.isscalar(stride) else stride
        pt, pb, pl, pr = (pad,) * 4 if np.isscalar(pad) else pad
        y = self.empty((n, k, (h - 1) * sh + kh - pt - pb, (wd - 1) * sw + kw - pl - pr), np.float32)
        _check(lib().exhip_deconv2d_f32(self.h, x.ptr, w.ptr, _ptr(bias), y.ptr, n, c, h, wd, k, kh, kw, sh, sw, pt, pb, pl, pr))
        return y

    def add_f16(self, a, b, relu=False):
        y = self.empty(a.shape, np.uint16)
        _check(lib().exhip_add_f16(self.h, a.ptr, b.ptr, y.ptr, ctypes.c_size_t(y.size), int(relu)))
        return y

    def relu_f16(self, x):
        y = self.empty(x.shape, np.uint16)
        _check(lib().exhip_relu_f16(self.h, x.ptr, y.ptr, ctypes.c_size_t(y.size)))
        return y

    def innerproduct_f32(self, x, w, bias=None):
        m = x.shape[0]
        k_in = x.size // m
        n_out = w.size // k_in
        y = self.empty((m, n_out, 1, 1), np.float32)
        _check(lib().exhip_innerproduct_f32(self.h, x.ptr, w.ptr, _ptr(bias), y.ptr, m, n_out, k_in))
        return y

    def innerproduct_f16(self, x, w, bias=None):
        m = x.shape[0]
        k_in = x.size // m
        n_out = w.size // k_in
        y = self.empty((m, n_out, 1, 1), np.uint16)
        _check(lib().exhip_innerproduct_f16(self.h, x.ptr, w.ptr, _ptr(bias), y.ptr, m, n_out, k_in))
        return y

    # ---- inner products in 8-bit floating point ----
    GATES = {"silu": 0, "gelu": 1, "sigmoid": 2, "relu": 3}

    def quantize_rows_f8(self, x, k=None, y=None, scale=None):
        """Rows x [m][stride] (float32, or halves as uint16 or float16) of k values: (codes [m][k up to 16], scales [k blocks][m])."""
        m, stride = x.shape
        k = stride if k is None else k
        if m > _MOST or stride > _MOST or k > _MOST:
            _size_refused(m, stride, k)
        if y is None:
            y = self.empty((m, pad_to(k, 16)), np.uint8)
        if scale is None:
            scale = self.empty((_blocks(k), m), np.float32)
        y_stride, scales = y.shape[1], -(-k // F8_BLOCK) * m
        if not (x.size >= (m - 1) * stride + k and x.char in _ROWS and y.size >= (m - 1) * y_stride + k and y.char in _CODES and scale.size >= scales and scale.char in _FLOATS):
            _refused(("x", x, (m - 1) * stride + k, _ROWS), ("y", y, (m - 1) * y_stride + k, _CODES), ("scale", scale, scales, _FLOATS))
        entry = (_lib or lib()).exhip_quantize_rows_f32_to_f8 if x.char == "f" else (_lib or lib()).exhip_quantize_rows_f16_to_f8
        rc = entry(self.h, x.ptr, stride, m, k, y.ptr, y_stride, scale.ptr)
        if rc:
            _check(rc)
        return y, scale

    def quantize_blocks_f8(self, w):
        """A float32 weight matrix [n][k]: (codes [n][k], scales [n blocks][k blocks])."""
        n, k = w.shape
        if n > _MOST or k > _MOST:
            _size_refused(n, k)
        _refused(("w", w, n * k, _FLOATS))
        y = self.empty((n, k), np.uint8)
        scale = self.empty((_blocks(n), _blocks(k)), np.float32)
        _check(lib().exhip_quantize_blocks_f32_to_f8(self.h, w.ptr, n, k, y.ptr, scale.ptr))
        return y, scale

    @staticmethod
    def f8_packed_bytes(n_out, k_in, gated=False):
        if n_out > _MOST or k_in > _MOST:
            _size_refused(n_out, k_in)
        nbytes = lib().exhip_f8_packed_bytes(int(n_out), int(k_in), int(gated))
        if nbytes == 0:
            raise ExhipError(f"exhip_f8_packed_bytes: {lib().exhip_last_error().decode()}")
        return nbytes

    def pack_f8_weights(self, n_out, k_in, w, w_up=None, packed=None):
        """Codes [n_out][k_in] in the product's order; with w_up those of a gated product, w the one in front of the activation."""
        nbytes = self.f8_packed_bytes(n_out, k_in, w_up is not None)
        _refused(("w", w, n_out * k_in, _CODES), ("w_up", w_up, n_out * k_in, _CODES), ("packed", packed, nbytes, _CODES))
        if packed is None:
            packed = self.empty((nbytes,), np.uint8)
        _check(lib().exhip_f8_pack_weights(self.h, n_out, k_in, w.ptr, _ptr(w_up), packed.ptr))
        return packed

    @staticmethod
    def f8_desc(m, n_out, k_in, x_stride=None, y_stride=None):
        x_stride, y_stride = pad_to(k_in, 16) if x_stride is None else x_stride, n_out if y_stride is None else y_stride
        if max(m, n_out, k_in, x_stride, y_stride) > _MOST:
            _size_refused(m, n_out, k_in, x_stride, y_stride)
        return F8Desc(m, n_out, k_in, x_stride, y_stride)

    def innerproduct_f8(self, d, x, x_scale, w, w_scale, bias=None, y_f32=None, y_f16=None, cut_sums=False):
        """cut_sums: the faster sums that keep 13 bits beneath the largest of eight products (exhip_innerproduct_cut_f8), for results in halves alone."""
        rows, scales, packed, w_scales, n, result, _ = d._counts or d.counts()
        if not (x.size >= rows and x.char in _CODES and x_scale.size >= scales and x_scale.char in _FLOATS and w.size >= packed and w.char in _CODES
                and w_scale.size >= w_scales and w_scale.char in _FLOATS and (bias is None or bias.size >= n and bias.char in _FLOATS)
                and (y_f32 is None or y_f32.size >= result and y_f32.char in _FLOATS) and (y_f16 is None or y_f16.size >= result and y_f16.char in _HALVES)):
            _refused(("x", x, rows, _CODES), ("x_scale", x_scale, scales, _FLOATS), ("w", w, packed, _CODES), ("w_scale", w_scale, w_scales, _FLOATS), ("bias", bias, n, _FLOATS),
                     ("y_f32", y_f32, result, _FLOATS), ("y_f16", y_f16, result, _HALVES))
        if cut_sums:
            if y_f32:
                raise ExhipError("cut sums are for results in halves alone")
            return _check(lib().exhip_innerproduct_cut_f8(self.h, ctypes.byref(d), x.ptr, x_scale.ptr, w.ptr, w_scale.ptr, _ptr(bias), _ptr(y_f16)))
        rc = (_lib or lib()).exhip_innerproduct_f8(self.h, ctypes.byref(d), x.ptr, x_scale.ptr, w.ptr, w_scale.ptr, bias and bias.ptr, y_f32 and y_f32.ptr, y_f16 and y_f16.ptr)
        if rc:
            _check(rc)

    def innerproduct_gated_f8(self, d, x, x_scale, w, w_scale_gate, w_scale_up, gate="silu", bias_gate=None, bias_up=None, y_f16=None, y_f8=None, y_scale=None,
                              cut_sums=False):
        """cut_sums: as of innerproduct_f8."""
        rows, scales, packed, w_scales, n, result, result_scales = d._counts or d.counts()
        if not (x.size >= rows and x.char in _CODES and x_scale.size >= scales and x_scale.char in _FLOATS and w.size >= 2 * packed and w.char in _CODES
                and w_scale_gate.size >= w_scales and w_scale_gate.char in _FLOATS and w_scale_up.size >= w_scales and w_scale_up.char in _FLOATS
                and _holds(bias_gate, n, _FLOATS) and _holds(bias_up, n, _FLOATS) and _holds(y_f16, result, _HALVES) and _holds(y_f8, result, _CODES)
                and _holds(y_scale, result_scales, _FLOATS)):
            _refused(("x", x, rows, _CODES), ("x_scale", x_scale, scales, _FLOATS), ("w", w, 2 * packed, _CODES), ("w_scale_gate", w_scale_gate, w_scales, _FLOATS),
                     ("w_scale_up", w_scale_up, w_scales, _FLOATS), ("bias_gate", bias_gate, n, _FLOATS), ("bias_up", bias_up, n, _FLOATS), ("y_f16", y_f16, result, _HALVES),
                     ("y_f8", y_f8, result, _CODES), ("y_scale", y_scale, result_scales, _FLOATS))
        if cut_sums:
            if y_f8 or y_scale:
                raise ExhipError("cut sums are for results in halves alone")
            return _check(lib().exhip_innerproduct_gated_cut_f8(self.h, ctypes.byref(d), self.GATES[gate], x.ptr, x_scale.ptr, w.ptr, w_scale_gate.ptr, w_scale_up.ptr,
                                                                _ptr(bias_gate), _ptr(bias_up), _ptr(y_f16)))
        rc = (_lib or lib()).exhip_innerproduct_gated_f8(self.h, ctypes.byref(d), self.GATES[gate], x.ptr, x_scale.ptr, w.ptr, w_scale_gate.ptr, w_scale_up.ptr,
                                                         bias_gate and bias_gate.ptr, bias_up and bias_up.ptr, y_f16 and y_f16.ptr, y_f8 and y_f8.ptr, y_scale and y_scale.ptr)
        if rc:
            _check(rc)

    # ---- inner products in 8-bit integers ----
    def quantize_rows_i8(self, x, k=None, y=None, scale=None):
        """Rows x [m][stride] (float32, or halves as uint16 or float16) of k values: (codes [m][k up to 16], scales [m])."""
        m, stride = x.shape
        k = stride if k is None else k
        if m > _MOST or stride > _MOST or k > _MOST:
            _size_refused(m, stride, k)
        if y is None:
            y = self.empty((m, pad_to(k, 16)), np.int8)
        if scale is None:
            scale = self.empty((m,), np.float32)
        y_stride = y.shape[1]
        if not (x.size >= (m - 1) * stride + k and x.char in _ROWS and y.size >= (m - 1) * y_stride + k and y.char in _CODES and scale.size >= m and scale.char in _FLOATS):
            _refused(("x", x, (m - 1) * stride + k, _ROWS), ("y", y, (m - 1) * y_stride + k, _CODES), ("scale", scale, m, _FLOATS))
        entry = (_lib or lib()).exhip_quantize_rows_f32_to_i8 if x.char == "f" else (_lib or lib()).exhip_quantize_rows_f16_to_i8
        rc = entry(self.h, x.ptr, stride, m, k, y.ptr, y_stride, scale.ptr)
        if rc:
            _check(rc)
        return y, scale

    @staticmethod
    @functools.lru_cache(maxsize=256)
    def i8_packed_bytes(n_out, k_in, gated=False, experts=1):
        if n_out > _MOST or k_in > _MOST or experts > _MOST:
            _size_refused(n_out, k_in, experts)
        nbytes = lib().exhip_i8_packed_bytes(int(experts), int(n_out), int(k_in), int(gated))
        if nbytes == 0:
            raise ExhipError(f"exhip_i8_packed_bytes: {lib().exhip_last_error().decode()}")
        return nbytes

    def pack_i8_weights(self, n_out, k_in, w, w_up=None, packed=None, experts=1):
        """Codes [experts][n_out][k_in] in the products' order; with w_up those of a gated product, w the one in front of the activation."""
        nbytes, count = self.i8_packed_bytes(n_out, k_in, w_up is not None, experts), experts * n_out * k_in
        _refused(("w", w, count, _CODES), ("w_up", w_up, count, _CODES), ("packed", packed, nbytes, _CODES))
        if packed is None:
            packed = self.empty((nbytes,), np.uint8)
        _check(lib().exhip_i8_pack_weights(self.h, experts, n_out, k_in, w.ptr, _ptr(w_up), packed.ptr))
        return packed

    @staticmethod
    def i8_desc(m, n_out, k_in, x_stride=None, y_stride=None):
        x_stride, y_stride = pad_to(k_in, 16) if x_stride is None else x_stride, n_out if y_stride is None else y_stride
        if max(m, n_out, k_in, x_stride, y_stride) > _MOST:
            _size_refused(m, n_out, k_in, x_stride, y_stride)
        return I8Desc(m, n_out, k_in, x_stride, y_stride)

    @staticmethod
    def _refused_i8(d, experts, gated, source, offsets, rows, x, x_scale, w, w_scale, w_scale_up, bias, bias_up, y_f32, y_f16):
        """Says which operand of a product is of another type or too small; `source` rows of the input."""
        _, _, packed, outputs, result = d.counts(experts, gated)
        scale, b = ("w_scale_gate", "bias_gate") if gated else ("w_scale", "bias")
        _refused(("x", x, (source - 1) * d.x_stride + d.k_in, _CODES), ("x_scale", x_scale, source, _FLOATS), ("w", w, packed, _CODES), (scale, w_scale, outputs, _FLOATS),
                 ("w_scale_up", w_scale_up, outputs, _FLOATS), (b, bias, outputs, _FLOATS), ("bias_up", bias_up, outputs, _FLOATS), ("y_f32", y_f32, result, _FLOATS),
                 ("y_f16", y_f16, result, _HALVES), ("offsets", offsets, experts + 1, _IDS), ("rows", rows, d.m, _IDS))

    def innerproduct_i8(self, d, x, x_scale, w, w_scale, bias=None, y_f32=None, y_f16=None):
        counts = d._counts
        if counts is None or counts[0] != (1, False):
            counts = d.counts()
        _, codes, packed, n, result = counts
        if not (x.size >= codes and x.char in _CODES and x_scale.size >= d.m and x_scale.char in _FLOATS and w.size >= packed and w.char in _CODES and w_scale.size >= n
                and w_scale.char in _FLOATS and (bias is None or bias.size >= n and bias.char in _FLOATS) and (y_f32 is None or y_f32.size >= result and y_f32.char in _FLOATS)
                and (y_f16 is None or y_f16.size >= result and y_f16.char in _HALVES)):
            self._refused_i8(d, 1, False, d.m, None, None, x, x_scale, w, w_scale, None, bias, None, y_f32, y_f16)
        rc = (_lib or lib()).exhip_innerproduct_i8(self.h, ctypes.byref(d), x.ptr, x_scale.ptr, w.ptr, w_scale.ptr, bias and bias.ptr, y_f32 and y_f32.ptr, y_f16 and y_f16.ptr)
        if rc:
            _check(rc)

    def innerproduct_gated_i8(self, d, x, x_scale, w, w_scale_gate, w_scale_up, gate="silu", bias_gate=None, bias_up=None, y_f32=None, y_f16=None):
        counts = d._counts
        if counts is None or counts[0] != (1, True):
            counts = d.counts(1, True)
        _, codes, packed, n, result = counts
        if not (x.size >= codes and x.char in _CODES and x_scale.size >= d.m and x_scale.char in _FLOATS and w.size >= packed and w.char in _CODES and w_scale_gate.size >= n
                and w_scale_gate.char in _FLOATS and w_scale_up.size >= n and w_scale_up.char in _FLOATS and _holds(bias_gate, n, _FLOATS) and _holds(bias_up, n, _FLOATS)
                and _holds(y_f32, result, _FLOATS) and _holds(y_f16, result, _HALVES)):
            self._refused_i8(d, 1, True, d.m, None, None, x, x_scale, w, w_scale_gate, w_scale_up, bias_gate, bias_up, y_f32, y_f16)
        rc = (_lib or lib()).exhip_innerproduct_gated_i8(self.h, ctypes.byref(d), self.GATES[gate], x.ptr, x_scale.ptr, w.ptr, w_scale_gate.ptr, w_scale_up.ptr,
                                                         bias_gate and bias_gate.ptr, bias_up and bias_up.ptr, y_f32 and y_f32.ptr, y_f16 and y_f16.ptr)
        if rc:
            _check(rc)

    # ---- by experts ----
    WEIGHTS = {"plain": 0, "log": 1, "log_normalized": 2}

    def group_rows(self, ids, experts, offsets=None, rows=None, places=None):
        """The choices ids [m][each] (int32) in order by expert: (offsets [experts + 1], rows [m * each], places [m][each])."""
        m, each = ids.shape
        if m > _MOST or each > _MOST or experts > _MOST:
            _size_refused(m, each, experts)
        offsets = self.empty((experts + 1,), np.int32) if offsets is None else offsets
        rows = self.empty((m * each,), np.int32) if rows is None else rows
        places = self.empty((m, each), np.int32) if places is None else places
        count = m * each
        if not (ids.size >= count and ids.char in _IDS and offsets.size > experts and offsets.char in _IDS and rows.size >= count and rows.char in _IDS and places.size >= count
                and places.char in _IDS):
            _refused(("ids", ids, m * each, _IDS), ("offsets", offsets, experts + 1, _IDS), ("rows", rows, m * each, _IDS), ("places", places, m * each, _IDS))
        rc = (_lib or lib()).exhip_group_rows(self.h, ids.ptr, m, each, experts, offsets.ptr, rows.ptr, places.ptr)
        if rc:
            _check(rc)
        return offsets, rows, places

    def innerproduct_grouped_i8(self, d, experts, offsets, x, x_scale, w, w_scale, bias=None, rows=None, x_rows=0, y_f32=None, y_f16=None):
        """d.m rows in order by expert; with `rows` they are those of the x_rows rows of x."""
        counts = d._counts
        if counts is None or counts[0] != (experts, False):
            counts = d.counts(experts, False)
        _, codes, packed, n, result = counts
        source = d.m
        if rows is not None:
            if x_rows > _MOST:
                _size_refused(x_rows)
            source, codes = x_rows, (x_rows - 1) * d.x_stride + d.k_in
        if not (x.size >= codes and x.char in _CODES and x_scale.size >= source and x_scale.char in _FLOATS and w.size >= packed and w.char in _CODES and w_scale.size >= n
                and w_scale.char in _FLOATS and _holds(bias, n, _FLOATS) and _holds(y_f32, result, _FLOATS) and _holds(y_f16, result, _HALVES)
                and offsets.size > experts and offsets.char in _IDS and _holds(rows, d.m, _IDS)):
            self._refused_i8(d, experts, False, source, offsets, rows, x, x_scale, w, w_scale, None, bias, None, y_f32, y_f16)
        rc = (_lib or lib()).exhip_innerproduct_grouped_i8(self.h, ctypes.byref(d), experts, offsets.ptr, rows and rows.ptr, x_rows, x.ptr, x_scale.ptr, w.ptr, w_scale.ptr,
                                                           bias and bias.ptr, y_f32 and y_f32.ptr, y_f16 and y_f16.ptr)
        if rc:
            _check(rc)

    def innerproduct_grouped_gated_i8(self, d, experts, offsets, x, x_scale, w, w_scale_gate, w_scale_up, gate="silu", bias_gate=None, bias_up=None, rows=None, x_rows=0,
                                      y_f32=None, y_f16=None):
        """d.m rows in order by expert; with `rows` they are those of the x_rows rows of x."""
        counts = d._counts
        if counts is None or counts[0] != (experts, True):
            counts = d.counts(experts, True)
        _, codes, packed, n, result = counts
        source = d.m
        if rows is not None:
            if x_rows > _MOST:
                _size_refused(x_rows)
            source, codes = x_rows, (x_rows - 1) * d.x_stride + d.k_in
        if not (x.size >= codes and x.char in _CODES and x_scale.size >= source and x_scale.char in _FLOATS and w.size >= packed and w.char in _CODES and w_scale_gate.size >= n
                and w_scale_gate.char in _FLOATS and w_scale_up.size >= n and w_scale_up.char in _FLOATS and _holds(bias_gate, n, _FLOATS) and _holds(bias_up, n, _FLOATS)
                and _holds(y_f32, result, _FLOATS) and _holds(y_f16, result, _HALVES) and offsets.size > experts and offsets.char in _IDS and _holds(rows, d.m, _IDS)):
            self._refused_i8(d, experts, True, source, offsets, rows, x, x_scale, w, w_scale_gate, w_scale_up, bias_gate, bias_up, y_f32, y_f16)
        rc = (_lib or lib()).exhip_innerproduct_grouped_gated_i8(self.h, ctypes.byref(d), self.GATES[gate], experts, offsets.ptr, rows and rows.ptr, x_rows, x.ptr, x_scale.ptr,
                                                                 w.ptr, w_scale_gate.ptr, w_scale_up.ptr, bias_gate and bias_gate.ptr, bias_up and bias_up.ptr,
                                                                 y_f32 and y_f32.ptr, y_f16 and y_f16.ptr)
        if rc:
            _check(rc)

    def combine_rows(self, z, places, weights, n=None, kind="plain", y_f32=None, y_f16=None):
        """For each row of places [m][each] the weighted sum of those rows of the halves z [rows][stride] of n values, into y_f32 or y_f16 [m][stride]."""
        (m, each), (z_rows, z_stride) = places.shape, z.shape
        n = z_stride if n is None else n
        if (y_f32 is None) == (y_f16 is None):
            raise ExhipError("one result: y_f32 or y_f16")
        y = y_f16 if y_f32 is None else y_f32
        y_stride = y.shape[1] if len(y.shape) > 1 else n
        if max(m, each, z_rows, z_stride, n, y_stride) > _MOST:
            _size_refused(m, each, z_rows, z_stride, n, y_stride)
        source, result, types = (z_rows - 1) * z_stride + n, (m - 1) * y_stride + n, _FLOATS if y_f16 is None else _HALVES
        if not (z.size >= source and z.char in _HALVES and places.size >= m * each and places.char in _IDS and weights.size >= m * each and weights.char in _FLOATS
                and y.size >= result and y.char in types):
            _refused(("z", z, source, _HALVES), ("places", places, m * each, _IDS), ("weights", weights, m * each, _FLOATS), ("y_f32" if y_f16 is None else "y_f16", y, result, types))
        entry = (_lib or lib()).exhip_combine_rows_f32 if y_f16 is None else (_lib or lib()).exhip_combine_rows_f16
        rc = entry(self.h, z.ptr, z_stride, z_rows, places.ptr, weights.ptr, self.WEIGHTS[kind], m, each, n, y.ptr, y_stride)
        if rc:
            _check(rc)

    # ---- answers ----
    @staticmethod
    @functools.lru_cache(maxsize=256)
    def log_probabilities_workspace(m, c, top=0):
        if m > _MOST or c > _MOST or top > _MOST:
            _size_refused(m, c, top)
        nbytes = lib().exhip_log_probabilities_workspace(int(m), int(c), int(top))
        if nbytes == 0:
            raise ExhipError(f"exhip_log_probabilities_workspace: {lib().exhip_last_error().decode()}")
        return nbytes

    def log_probabilities(self, x, c=None, ids=None, top=0, log_p=None, entropy=None, top_ids=None, top_log_p=None, workspace=None):
        """Of rows x [m][stride] (float32, or halves as uint16 or float16) of c values: the log probabilities of ids [m][n] (int32), the entropy, the `top`
        largest classes and their log probabilities, into the given arrays. Without a workspace it makes one and waits for the results; a recorded run is
        given one."""
        m, stride = x.shape
        c = stride if c is None else c
        n_ids = ids.shape[1] if ids is not None else 0
        if stride > _MOST or n_ids > _MOST:
            _size_refused(stride, n_ids)
        nbytes = self.log_probabilities_workspace(m, c, top)
        if not (_holds(x, (m - 1) * stride + c, _ROWS) and _holds(ids, m * n_ids, _IDS) and _holds(log_p, m * n_ids, _FLOATS) and _holds(entropy, m, _FLOATS)
                and _holds(top_ids, m * top, _IDS) and _holds(top_log_p, m * top, _FLOATS)):
            _refused(("x", x, (m - 1) * stride + c, _ROWS), ("ids", ids, m * n_ids, _IDS), ("log_p", log_p, m * n_ids, _FLOATS), ("entropy", entropy, m, _FLOATS),
                     ("top_ids", top_ids, m * top, _IDS), ("top_log_p", top_log_p, m * top, _FLOATS))
        if workspace is not None and not isinstance(workspace, _Inside) and workspace.size * workspace.dtype.itemsize < nbytes:
            raise ExhipError(f"workspace has {workspace.size * workspace.dtype.itemsize} bytes, the call takes {nbytes}")
        own = self.empty((nbytes,), np.uint8) if workspace is None else None
        entry = lib().exhip_log_probabilities_f32 if x.char == "f" else lib().exhip_log_probabilities_f16
        rc = entry(self.h, x.ptr, stride, m, c, _ptr(ids), n_ids, _ptr(log_p), _ptr(entropy), top, _ptr(top_ids), _ptr(top_log_p),
                   (own if workspace is None else workspace).ptr)
        if own is not None:
            own.free()
        _check(rc)

    def stem_f16(self, d, x, mean, factor, wp, bias, y):
        """The status: 0, or EXHIP_ERR_UNSUPPORTED where the layers run by themselves."""
        rc = lib().exhip_stem_f16(self.h, ctypes.byref(d), x.ptr, _ptr(mean), _ptr(factor), wp.ptr, _ptr(bias), y.ptr)
        return rc if rc == ERR_UNSUPPORTED else _check(rc) or 0

    def stem_i8(self, d, x, mean, factor, fs_in, wp, scale, bias, y_i8, y_f32=None):
        """As stem_f16."""
        rc = lib().exhip_stem_i8(self.h, ctypes.byref(d), x.ptr, _ptr(mean), _ptr(factor), ctypes.c_float(fs_in), wp.ptr, scale.ptr, _ptr(bias),
                                 _ptr(y_i8), _ptr(y_f32))
        return rc if rc == ERR_UNSUPPORTED else _check(rc) or 0

    def conv2d_i8_maxpool2x2(self, d, pool_oh, pool_ow, x, wp, scale, bias=None, y_i8=None, y_f32=None):
        """As stem_f16."""
        rc = lib().exhip_conv2d_i8_maxpool2x2(self.h, ctypes.byref(d), pool_oh, pool_ow, x.ptr, wp.ptr, scale.ptr, _ptr(bias), _ptr(y_i8), _ptr(y_f32))
        return rc if rc == ERR_UNSUPPORTED else _check(rc) or 0
