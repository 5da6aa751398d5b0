"""ctypes binding of libien_hip.so, the MI355X backend's C ABI
(include/ien_hip.h), for the tests and the benchmark.

Device buffers are torch tensors on the GPU (plumbing only: the kernels are
the library's); the library runs on torch's current stream, so torch events
and synchronisation order with it.  Nothing here falls back to the CPU: a
missing or unloadable library raises.
"""

import ctypes
import pathlib
import struct

HERE = pathlib.Path(__file__).resolve().parent
LIB_PATH = HERE / "libien_hip.so"

OK, ERR_IO, ERR_WEIGHTS, ERR_INPUT, ERR_CANCELLED, ERR_GPU = range(6)
W_F32, W_F16 = 0, 1
PAD_ZERO, PAD_REFLECT = 0, 1
TAPS_CONV, TAPS_OFFSETS = 0, 1
INPUT_ROWS, INPUT_IMAGE = 0, 1
NHWC, NCHW = 0, 1
ACT_NONE, ACT_RELU, ACT_GELU, ACT_PRELU, ACT_SIGMOID, ACT_SILU = range(6)
OUT_F16, OUT_F32 = 0, 1
MODEL_REALESRGAN, MODEL_SCUNET, MODEL_LAMA, MODEL_BIREFNET = 0, 1, 2, 3
SCORE_SOFTMAX, SCORE_SIGMOID = 0, 1

# Every symbol include/ien_hip.h declares.
EXPORTS = (
    "ien_last_error", "ien_open", "ien_close", "ien_device_name", "ien_stream", "ien_set_stream",
    "ien_alloc", "ien_free", "ien_upload", "ien_download", "ien_sync",
    "ien_floats_to_halves", "ien_halves_to_floats",
    "ien_matrix_new", "ien_matrix_free", "ien_multiply", "ien_multiply_ex", "ien_conv3",
    "ien_conv3_pair", "ien_conv3_chain", "ien_conv3_chain_status", "ien_measure_mfma",
    "ien_layer_norm", "ien_gelu", "ien_sigmoid", "ien_pixel_shuffle_add", "ien_depthwise",
    "ien_model_load", "ien_model_from_tensors", "ien_model_free", "ien_model_run",
    "ien_model_run_device", "ien_model_status", "ien_model_set_graph", "ien_model_run_tiled", "ien_model_run_u8",
    "ien_bytes_to_floats", "ien_floats_to_bytes", "ien_mask_bytes", "ien_normalize_bytes",
    "ien_composite_bytes",
    "ien_window_count", "ien_position_bias", "ien_bias_tables", "ien_window_gather",
    "ien_window_attention", "ien_window_scatter_add", "ien_swin_new", "ien_swin_free", "ien_swin_run",
    "ien_swin_run_static",
    "ien_resize", "ien_pad_image", "ien_crop", "ien_gather_2x2", "ien_scatter_2x2", "ien_add",
    "ien_fourier_new", "ien_fourier_free", "ien_fourier_half", "ien_fourier_forward",
    "ien_fourier_inverse", "ien_spectral_new", "ien_spectral_free", "ien_spectral_work",
    "ien_spectral_run",
    "ien_rows8_stride", "ien_rows8_scale_stride", "ien_quantize8", "ien_dequantize8", "ien_matrix8_new",
    "ien_matrix8_free", "ien_multiply8", "ien_group_norm", "ien_group_norm8",
    "ien_rms_norm", "ien_routes_ints", "ien_routes_order", "ien_route", "ien_routes_plan", "ien_experts8_new",
    "ien_experts8_free", "ien_experts_in8", "ien_experts_parts", "ien_experts_out8",
    "ien_experts_out8_ex",
)


class Windows(ctypes.Structure):
    """ien_windows: a Swin block's windows over a height x width token map."""
    _fields_ = [("window", ctypes.c_int), ("shift", ctypes.c_int), ("height", ctypes.c_int),
                ("width", ctypes.c_int)]


POS_SCUNET, POS_SWIN = 0, 1
PAD_REPLICATE, PAD_SYMMETRIC_MASKED = 0, 1
ORDER_ROW_MAJOR, ORDER_COLUMN_MAJOR = 0, 1


class SwinWeights(ctypes.Structure):
    """ien_swin_weights (host f32 pointers)."""
    _fields_ = [("c", ctypes.c_int), ("window", ctypes.c_int), ("shift", ctypes.c_int),
                ("masked", ctypes.c_float)] + [
        (name, ctypes.c_void_p) for name in (
            "ln1_gamma", "ln1_beta", "qkv_w", "qkv_b", "position", "proj_w", "proj_b", "ln2_gamma",
            "ln2_beta", "fc1_w", "fc1_b", "fc2_w", "fc2_b")]


class IenError(RuntimeError):
    def __init__(self, status, message):
        super().__init__(message)
        self.status = status


class Input(ctypes.Structure):
    _fields_ = [
        ("kind", ctypes.c_int),
        ("data", ctypes.c_void_p),
        ("height", ctypes.c_size_t),
        ("width", ctypes.c_size_t),
        ("channels", ctypes.c_size_t),
        ("stride", ctypes.c_size_t),
        ("layout", ctypes.c_int),
        ("taps", ctypes.c_int),
        ("size", ctypes.c_size_t),
        ("step", ctypes.c_size_t),
        ("pad", ctypes.c_int),
        ("offsets", (ctypes.c_size_t * 2) * 4),
        ("count", ctypes.c_size_t),
    ]


class Output(ctypes.Structure):
    _fields_ = [
        ("data", ctypes.c_void_p),
        ("stride", ctypes.c_size_t),
        ("layout", ctypes.c_int),
        ("type", ctypes.c_int),
    ]


class Rows8Struct(ctypes.Structure):
    """ien_rows8."""
    _fields_ = [("data", ctypes.c_void_p), ("stride", ctypes.c_size_t), ("scales", ctypes.c_void_p),
                ("scale_stride", ctypes.c_size_t)]


class Input8(ctypes.Structure):
    """ien_input8."""
    _fields_ = [("kind", ctypes.c_int), ("map", Rows8Struct), ("images", ctypes.c_size_t),
                ("height", ctypes.c_size_t), ("width", ctypes.c_size_t), ("step", ctypes.c_size_t),
                ("fast", ctypes.c_int)]


class RoutesStruct(ctypes.Structure):
    """ien_routes."""
    _fields_ = [("tokens", ctypes.c_size_t), ("experts", ctypes.c_size_t), ("top", ctypes.c_size_t),
                ("index", ctypes.c_void_p), ("weight", ctypes.c_void_p), ("plan", ctypes.c_void_p)]


class Router(ctypes.Structure):
    """ien_router."""
    _fields_ = [("score", ctypes.c_int), ("bias", ctypes.c_void_p), ("groups", ctypes.c_size_t), ("kept", ctypes.c_size_t),
                ("group_top", ctypes.c_size_t), ("renormalise", ctypes.c_int), ("scale", ctypes.c_float)]


class Tensor(ctypes.Structure):
    _fields_ = [
        ("name", ctypes.c_char_p),
        ("rank", ctypes.c_size_t),
        ("dims", ctypes.c_size_t * 4),
        ("values", ctypes.c_void_p),
    ]


PROGRESS = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_float, ctypes.c_void_p)

_lib = None


def load():
    """The library, loaded once; raises if it is not built."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise OSError(f"{LIB_PATH} is not built: run __graft_entry__.build()")
        L = ctypes.CDLL(str(LIB_PATH))
        vp, sz, st, i = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_int
        L.ien_last_error.restype = ctypes.c_char_p
        L.ien_open.argtypes = [i, ctypes.POINTER(vp)]
        L.ien_close.argtypes = [vp]
        L.ien_close.restype = None
        L.ien_device_name.argtypes = [vp]
        L.ien_device_name.restype = ctypes.c_char_p
        L.ien_stream.argtypes = [vp]
        L.ien_stream.restype = vp
        L.ien_set_stream.argtypes = [vp, vp]
        L.ien_alloc.argtypes = [vp, sz, ctypes.POINTER(vp)]
        L.ien_free.argtypes = [vp, vp]
        L.ien_upload.argtypes = [vp, vp, vp, sz]
        L.ien_download.argtypes = [vp, vp, vp, sz]
        L.ien_sync.argtypes = [vp]
        L.ien_floats_to_halves.argtypes = [vp, vp, vp, sz]
        L.ien_halves_to_floats.argtypes = [vp, vp, vp, sz]
        L.ien_matrix_new.argtypes = [vp, vp, i, sz, sz, vp, ctypes.POINTER(vp)]
        L.ien_matrix_free.argtypes = [vp]
        L.ien_matrix_free.restype = None
        L.ien_multiply.argtypes = [vp, ctypes.POINTER(Input), sz, sz, vp, vp, sz, i, i]
        L.ien_multiply_ex.argtypes = [vp, ctypes.POINTER(Input), sz, sz, vp, ctypes.POINTER(Output), i, vp, i]
        L.ien_conv3.argtypes = [vp, ctypes.POINTER(Input), vp, vp, sz, i, i, vp]
        L.ien_conv3_pair.argtypes = [vp, vp, vp, sz, sz, vp, vp, vp, vp]
        L.ien_conv3_chain.argtypes = [vp, vp, vp, sz, sz, sz, ctypes.POINTER(vp), ctypes.POINTER(vp),
                                      ctypes.POINTER(vp)]
        L.ien_conv3_chain_status.argtypes = [vp]
        L.ien_measure_mfma.argtypes = [vp, i, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_double)]
        L.ien_layer_norm.argtypes = [vp, vp, sz, sz, sz, vp, vp]
        L.ien_gelu.argtypes = [vp, vp, sz]
        L.ien_sigmoid.argtypes = [vp, vp, sz]
        L.ien_pixel_shuffle_add.argtypes = [vp, vp, sz, vp, sz, sz, vp]
        L.ien_depthwise.argtypes = [vp, vp, sz, sz, sz, i, vp, sz, vp, vp]
        L.ien_model_load.argtypes = [vp, i, ctypes.c_char_p, ctypes.POINTER(vp)]
        L.ien_model_from_tensors.argtypes = [vp, i, ctypes.POINTER(Tensor), sz, ctypes.POINTER(vp)]
        L.ien_model_free.argtypes = [vp]
        L.ien_model_free.restype = None
        L.ien_model_run.argtypes = [vp, vp, vp, sz, sz, vp, vp, vp]
        L.ien_model_run_tiled.argtypes = [vp, vp, sz, sz, sz, sz, vp, vp, vp]
        L.ien_model_run_u8.argtypes = [vp, vp, vp, sz, sz, vp, vp, vp]
        L.ien_bytes_to_floats.argtypes = [vp, vp, vp, sz]
        L.ien_floats_to_bytes.argtypes = [vp, vp, vp, sz]
        L.ien_mask_bytes.argtypes = [vp, vp, vp, sz]
        L.ien_normalize_bytes.argtypes = [vp, vp, sz, vp, vp, vp]
        L.ien_composite_bytes.argtypes = [vp, vp, vp, vp, sz, vp]
        L.ien_model_run_device.argtypes = [vp, vp, vp, sz, sz, vp]
        L.ien_model_status.argtypes = [vp]
        L.ien_model_set_graph.argtypes = [vp, i]
        wp = ctypes.POINTER(Windows)
        L.ien_window_count.argtypes = [wp]
        L.ien_window_count.restype = ctypes.c_long
        L.ien_position_bias.argtypes = [vp, i, i, i, vp]
        L.ien_bias_tables.argtypes = [vp, i, i, i, ctypes.c_float, vp]
        L.ien_bias_tables.restype = i
        L.ien_window_gather.argtypes = [vp, wp, vp, sz, i, vp, vp, vp]
        L.ien_window_attention.argtypes = [vp, wp, vp, i, vp, vp]
        L.ien_window_scatter_add.argtypes = [vp, wp, vp, i, vp, sz]
        L.ien_swin_new.argtypes = [vp, ctypes.POINTER(SwinWeights), ctypes.POINTER(vp)]
        L.ien_swin_free.argtypes = [vp]
        L.ien_swin_free.restype = None
        L.ien_swin_run.argtypes = [vp, vp, sz, i, i]
        L.ien_swin_run_static.argtypes = [vp, vp, sz, i, i]
        L.ien_resize.argtypes = [vp, vp, sz, sz, sz, sz, vp, sz, sz, sz, i, i]
        L.ien_pad_image.argtypes = [vp, i, vp, vp, sz, sz, sz, vp, sz]
        L.ien_crop.argtypes = [vp, vp, sz, sz, sz, sz, sz, vp]
        L.ien_gather_2x2.argtypes = [vp, vp, sz, sz, sz, sz, i, vp]
        L.ien_scatter_2x2.argtypes = [vp, vp, sz, sz, sz, sz, vp, sz]
        L.ien_add.argtypes = [vp, vp, vp, sz]
        L.ien_fourier_new.argtypes = [vp, sz, sz, ctypes.POINTER(vp)]
        L.ien_fourier_free.argtypes = [vp]
        L.ien_fourier_free.restype = None
        L.ien_fourier_half.argtypes = [vp]
        L.ien_fourier_half.restype = sz
        L.ien_fourier_forward.argtypes = [vp, vp, sz, sz, vp, vp]
        L.ien_fourier_inverse.argtypes = [vp, vp, sz, vp, vp, sz]
        L.ien_spectral_new.argtypes = [vp, sz, sz, ctypes.POINTER(vp)]
        L.ien_spectral_free.argtypes = [vp]
        L.ien_spectral_free.restype = None
        L.ien_spectral_work.argtypes = [vp]
        L.ien_spectral_work.restype = sz
        L.ien_spectral_run.argtypes = [vp, vp, sz, vp, vp, vp, vp, vp, vp, sz]
        fl = ctypes.c_float
        L.ien_rows8_stride.argtypes = [sz]
        L.ien_rows8_stride.restype = sz
        L.ien_rows8_scale_stride.argtypes = [sz]
        L.ien_rows8_scale_stride.restype = sz
        L.ien_quantize8.argtypes = [vp, vp, i, sz, sz, sz, vp]
        L.ien_dequantize8.argtypes = [vp, vp, sz, sz, vp, i, sz]
        L.ien_matrix8_new.argtypes = [vp, vp, i, sz, sz, sz, vp, ctypes.POINTER(vp)]
        L.ien_matrix8_free.argtypes = [vp]
        L.ien_matrix8_free.restype = None
        L.ien_multiply8.argtypes = [vp, vp, sz, sz, vp, vp, i, vp, sz]
        L.ien_group_norm.argtypes = [vp, vp, i, sz, sz, sz, sz, sz, vp, vp, fl, i, vp, i, sz]
        L.ien_group_norm8.argtypes = [vp, vp, i, sz, sz, sz, sz, sz, vp, vp, fl, i, vp]
        L.ien_rms_norm.argtypes = [vp, vp, i, sz, sz, sz, vp, i, sz, vp, sz, vp, fl, vp, i, sz, vp]
        L.ien_routes_ints.argtypes = [sz, sz, sz]
        L.ien_routes_ints.restype = sz
        L.ien_routes_order.argtypes = [sz]
        L.ien_routes_order.restype = sz
        L.ien_route.argtypes = [vp, vp, i, sz, vp, vp]
        L.ien_routes_plan.argtypes = [vp, vp]
        L.ien_experts8_new.argtypes = [vp, vp, i, sz, sz, sz, i, vp, ctypes.POINTER(vp)]
        L.ien_experts8_free.argtypes = [vp]
        L.ien_experts8_free.restype = None
        L.ien_experts_in8.argtypes = [vp, vp, vp, vp, i, i, vp]
        L.ien_experts_parts.argtypes = [vp, vp]
        L.ien_experts_parts.restype = sz
        L.ien_experts_out8.argtypes = [vp, vp, vp, vp, i, vp, vp, sz, vp]
        L.ien_experts_out8_ex.argtypes = [vp, vp, vp, vp, i, vp, i, vp, sz, vp, i, sz, vp]
        for name in EXPORTS:
            getattr(L, name)
        _lib = L
    return _lib


def check(status):
    if status != OK:
        raise IenError(status, load().ien_last_error().decode(errors="replace"))


def _ptr(t):
    """Device pointer of a torch tensor, or None."""
    return None if t is None else ctypes.c_void_p(t.data_ptr())


class Context:
    """ien_ctx on one device.  The context's own (non-blocking) HIP stream
    becomes torch's current stream, so torch's copies, fills and events are
    ordered with the library's launches; when it closes, that of the context
    opened last of those still open (or the default stream) takes its place."""

    _open = []

    def __init__(self, device=0):
        import torch

        L = load()
        h = ctypes.c_void_p()
        check(L.ien_open(device, ctypes.byref(h)))
        self.h = h
        self.device = device
        self.stream = torch.cuda.ExternalStream(L.ien_stream(h), device=torch.device("cuda", device))
        torch.cuda.set_stream(self.stream)
        Context._open.append(self)

    @property
    def name(self):
        return load().ien_device_name(self.h).decode()

    def close(self):
        if self.h:
            import torch

            torch.cuda.synchronize(self.device)
            Context._open.remove(self)
            if torch.cuda.current_stream(self.device) == self.stream:
                left = [c.stream for c in Context._open if c.device == self.device]
                torch.cuda.set_stream(left[-1] if left else torch.cuda.default_stream(self.device))
            load().ien_close(self.h)
            self.h = None

    def sync(self):
        check(load().ien_sync(self.h))


def settle(ctx):
    """Waits for torch's current stream unless it is the context's: of a tensor that
    torch has just made, fills and what lay in its memory before may be under way
    there, and the context's launches do not follow them."""
    import torch

    stream = torch.cuda.current_stream(ctx.device)
    if stream.cuda_stream != load().ien_stream(ctx.h):
        stream.synchronize()


class Matrix:
    """gemm.rs Matrix::new: host weights k x n (numpy f32 or f16) + bias."""

    def __init__(self, ctx, w, bias=None):
        import numpy as np

        w = np.ascontiguousarray(w)
        wtype = W_F16 if w.dtype == np.float16 else W_F32
        if wtype == W_F32:
            w = np.ascontiguousarray(w, dtype=np.float32)
        k, n = w.shape
        b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float32)
        h = ctypes.c_void_p()
        check(load().ien_matrix_new(ctx.h, w.ctypes.data_as(ctypes.c_void_p), wtype, k, n,
                                    None if b is None else b.ctypes.data_as(ctypes.c_void_p),
                                    ctypes.byref(h)))
        self.h, self.k, self.n, self.ctx = h, k, n, ctx

    def free(self):
        if self.h:
            load().ien_matrix_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def image_input(x, height, width, channels, stride=None, layout=NHWC, size=3, step=1, pad=PAD_ZERO,
                offsets=None):
    s = Input()
    s.kind = INPUT_IMAGE
    s.data = x.data_ptr()
    s._tensor = x  # the descriptor holds a raw pointer: keep its storage alive
    s.height, s.width, s.channels = height, width, channels
    s.stride = stride if stride is not None else (channels if layout == NHWC else height * width)
    s.layout = layout
    if offsets is None:
        s.taps, s.size, s.step, s.pad = TAPS_CONV, size, step, pad
    else:
        s.taps, s.count = TAPS_OFFSETS, len(offsets)
        for j, (dy, dx) in enumerate(offsets):
            s.offsets[j][0], s.offsets[j][1] = dy, dx
    return s


def rows_input(x, stride):
    s = Input()
    s.kind = INPUT_ROWS
    s.data = x.data_ptr()
    s._tensor = x  # the descriptor holds a raw pointer: keep its storage alive
    s.stride = stride
    return s


def multiply_ex(ctx, inp, row0, rows, matrix, out, out_stride, layout=NHWC, out_f32=False, act=ACT_NONE,
                slope=None, accumulate=False):
    o = Output()
    o.data = out.data_ptr()
    o.stride = out_stride
    o.layout = layout
    o.type = OUT_F32 if out_f32 else OUT_F16
    check(load().ien_multiply_ex(ctx.h, ctypes.byref(inp), row0, rows, matrix.h, ctypes.byref(o), act,
                                 _ptr(slope), int(accumulate)))


def multiply(ctx, inp, row0, rows, matrix, out, stride, act=ACT_NONE, accumulate=False):
    check(load().ien_multiply(ctx.h, ctypes.byref(inp), row0, rows, matrix.h, _ptr(out), stride, act,
                              int(accumulate)))


def conv3(ctx, inp, matrix, out, stride, accumulate=False, finish=ACT_NONE, slope=None):
    check(load().ien_conv3(ctx.h, ctypes.byref(inp), matrix.h, _ptr(out), stride, int(accumulate), finish,
                           _ptr(slope)))


def conv3_pair(ctx, x, y, height, width, m1, slope1, m2, slope2):
    """Two 3x3 64->64 PReLU layers in one launch, x -> y (H x W x 64 f16)."""
    check(load().ien_conv3_pair(ctx.h, _ptr(x), _ptr(y), height, width, m1.h, _ptr(slope1), m2.h,
                                _ptr(slope2)))


def conv3_chain(ctx, a, b, height, width, matrices, slopes):
    """len(matrices) / 2 pairs of 3x3 64->64 PReLU layers in one launch; the
    input in a, b a second map; returns the tensor (a or b) holding the
    output."""
    n = len(matrices)
    w = (ctypes.c_void_p * n)(*[m.h for m in matrices])
    s = (ctypes.c_void_p * n)(*[_ptr(x) for x in slopes])
    out = ctypes.c_void_p()
    check(load().ien_conv3_chain(ctx.h, _ptr(a), _ptr(b), height, width, n // 2, w, s, ctypes.byref(out)))
    return a if out.value == a.data_ptr() else b


def conv3_chain_status(ctx):
    check(load().ien_conv3_chain_status(ctx.h))


def measure_mfma(ctx, iters):
    """(sustained f16 MFMA TFLOP/s, ms) of a register-only MFMA loop on every SIMD."""
    tf, ms = ctypes.c_double(), ctypes.c_double()
    check(load().ien_measure_mfma(ctx.h, iters, ctypes.byref(tf), ctypes.byref(ms)))
    return tf.value, ms.value


def floats_to_halves(ctx, src, dst):
    check(load().ien_floats_to_halves(ctx.h, _ptr(src), _ptr(dst), src.numel()))


def halves_to_floats(ctx, src, dst):
    check(load().ien_halves_to_floats(ctx.h, _ptr(src), _ptr(dst), src.numel()))


def layer_norm(ctx, x, rows, c, stride, gamma, beta):
    check(load().ien_layer_norm(ctx.h, _ptr(x), rows, c, stride, _ptr(gamma), _ptr(beta)))


def gelu(ctx, x):
    check(load().ien_gelu(ctx.h, _ptr(x), x.numel()))


def sigmoid(ctx, x):
    check(load().ien_sigmoid(ctx.h, _ptr(x), x.numel()))


def pixel_shuffle_add(ctx, last, last_stride, image, width, height, out):
    check(load().ien_pixel_shuffle_add(ctx.h, _ptr(last), last_stride, _ptr(image), width, height, _ptr(out)))


def depthwise(ctx, x, height, width, channels, layout, w, size, bias, y):
    check(load().ien_depthwise(ctx.h, _ptr(x), height, width, channels, layout, _ptr(w), size, _ptr(bias),
                               _ptr(y)))


def windows(window, shift, height, width):
    return Windows(window, shift, height, width)


def window_count(w):
    n = load().ien_window_count(ctypes.byref(w))
    if n < 0:
        check(ERR_INPUT)
    return n


def _np_ptr(a):
    return ctypes.c_void_p(a.ctypes.data)


def position_bias(table, heads, window, layout):
    """[heads, N, N] from a SCUNet [heads, 2W-1, 2W-1] or Swin [(2W-1)^2, heads] table (host)."""
    import numpy as np

    table = np.ascontiguousarray(table, dtype=np.float32)
    out = np.zeros((heads, window * window, window * window), np.float32)
    check(load().ien_position_bias(_np_ptr(table), heads, window, layout, _np_ptr(out)))
    return out


def bias_tables(position, window, shift, masked):
    """[classes, heads, N, N] (host): swin.rs bias_tables."""
    import numpy as np

    position = np.ascontiguousarray(position, dtype=np.float32)
    heads, n = position.shape[0], window * window
    out = np.zeros((4, heads, n, n), np.float32)
    k = load().ien_bias_tables(_np_ptr(position), heads, window, shift, masked, _np_ptr(out))
    if k < 0:
        check(ERR_INPUT)
    return out[:k]


def window_gather(ctx, w, map_, stride, c, gamma, beta, tokens):
    check(load().ien_window_gather(ctx.h, ctypes.byref(w), _ptr(map_), stride, c, _ptr(gamma), _ptr(beta),
                                   _ptr(tokens)))


def window_attention(ctx, w, qkv, c, tables, out):
    check(load().ien_window_attention(ctx.h, ctypes.byref(w), _ptr(qkv), c, _ptr(tables), _ptr(out)))


def window_scatter_add(ctx, w, rows, c, map_, stride):
    check(load().ien_window_scatter_add(ctx.h, ctypes.byref(w), _ptr(rows), c, _ptr(map_), stride))


def resize(ctx, src, sh, sw, src_stride, c, dst, dh, dw, dst_stride, out_f32=False, add=False):
    check(load().ien_resize(ctx.h, _ptr(src), sh, sw, src_stride, c, _ptr(dst), dh, dw, dst_stride,
                            OUT_F32 if out_f32 else OUT_F16, int(add)))


def pad_image(ctx, mode, image, mask, width, height, multiple, out, stride):
    check(load().ien_pad_image(ctx.h, mode, _ptr(image), _ptr(mask), width, height, multiple, _ptr(out),
                               stride))


def crop(ctx, map_, map_width, stride, width, height, channels, out):
    check(load().ien_crop(ctx.h, _ptr(map_), map_width, stride, width, height, channels, _ptr(out)))


def gather_2x2(ctx, map_, height, width, c, stride, order, rows):
    check(load().ien_gather_2x2(ctx.h, _ptr(map_), height, width, c, stride, order, _ptr(rows)))


def scatter_2x2(ctx, rows, row_stride, height, width, c, map_, stride):
    check(load().ien_scatter_2x2(ctx.h, _ptr(rows), row_stride, height, width, c, _ptr(map_), stride))


def add(ctx, x, y):
    check(load().ien_add(ctx.h, _ptr(x), _ptr(y), x.numel()))


class Fourier:
    """ien_fourier: the 2-D real transforms of height x width maps."""

    def __init__(self, ctx, height, width):
        h = ctypes.c_void_p()
        check(load().ien_fourier_new(ctx.h, height, width, ctypes.byref(h)))
        self.h, self.height, self.width = h, height, width
        self.half = load().ien_fourier_half(h)

    def forward(self, x, stride, channels, work, spectrum):
        check(load().ien_fourier_forward(self.h, _ptr(x), stride, channels, _ptr(work), _ptr(spectrum)))

    def inverse(self, spectrum, channels, work, out, stride):
        check(load().ien_fourier_inverse(self.h, _ptr(spectrum), channels, _ptr(work), _ptr(out), stride))

    def free(self):
        if self.h:
            load().ien_fourier_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class Spectral:
    """ien_spectral: LaMa's FFC spectral branch (spectral_in product, rfftn,
    fourier product, irfftn added, spectral_out product accumulated with
    ReLU) for height x width maps of sides up to 64."""

    def __init__(self, ctx, height, width):
        h = ctypes.c_void_p()
        check(load().ien_spectral_new(ctx.h, height, width, ctypes.byref(h)))
        self.h, self.height, self.width = h, height, width
        self.work_floats = load().ien_spectral_work(h)

    def run(self, x, stride, spectral_in, fourier, spectral_out, spectral, work, out, out_stride):
        check(load().ien_spectral_run(self.h, _ptr(x), stride, spectral_in.h, fourier.h,
                                      spectral_out.h, _ptr(spectral), _ptr(work), _ptr(out),
                                      out_stride))

    def free(self):
        if self.h:
            load().ien_spectral_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class Swin:
    """ien_swin: one Swin transformer block (attend then MLP, in place).
    `weights`: dict of host arrays ln1_gamma, ln1_beta, qkv_w (c x 3c),
    qkv_b, position ([heads, N, N]), proj_w, proj_b, ln2_gamma, ln2_beta,
    fc1_w (c x 4c), fc1_b, fc2_w (4c x c), fc2_b."""

    def __init__(self, ctx, c, window, shift, masked, weights):
        import numpy as np

        keep = {k: np.ascontiguousarray(v, dtype=np.float32) for k, v in weights.items()}
        sw = SwinWeights(c, window, shift, masked)
        for name, _ in SwinWeights._fields_[4:]:
            setattr(sw, name, keep[name].ctypes.data)
        h = ctypes.c_void_p()
        check(load().ien_swin_new(ctx.h, ctypes.byref(sw), ctypes.byref(h)))
        self.h = h

    def run(self, map_, stride, height, width):
        check(load().ien_swin_run(self.h, _ptr(map_), stride, height, width))

    def run_static(self, map_, stride, height, width):
        """ien_swin_run_static: the same block with the library's static
        scratch (allocates nothing)."""
        check(load().ien_swin_run_static(self.h, _ptr(map_), stride, height, width))

    def free(self):
        if self.h:
            load().ien_swin_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class Rows8:
    """ien_rows8 over torch tensors: `rows` rows of k values in 8 bits (data:
    uint8 [rows, at least ien_rows8_stride(k)], scales: uint8 [rows, at least
    ien_rows8_scale_stride(k)]), made here unless given.  The tensors stay this
    object's (their addresses are read once, here); another Rows8 takes other
    ones, views of these among them."""

    def __init__(self, rows, k, data=None, scales=None, device="cuda"):
        import torch

        L = load()
        widths = L.ien_rows8_stride(k), L.ien_rows8_scale_stride(k)
        if data is None:
            data = torch.empty(rows, widths[0], dtype=torch.uint8, device=device)
        if scales is None:
            scales = torch.empty(rows, widths[1], dtype=torch.uint8, device=data.device)
        for t, width in zip((data, scales), widths):
            if t.dtype != torch.uint8 or t.dim() != 2 or t.shape[0] != rows or (t.shape[1] > 1 and t.stride(1) != 1):
                raise ValueError("rows in 8 bits are uint8 tensors of rows x bytes")
            if rows and t.shape[1] < width:
                raise ValueError(f"rows of {k} values in 8 bits take {width} bytes, not {t.shape[1]}")
        if data.device != scales.device:
            raise ValueError(f"rows in 8 bits on {data.device} and {scales.device}")
        self.rows, self.k, self._data, self._scales = rows, k, data, scales
        self._fields = data.data_ptr(), _row_stride(data), scales.data_ptr(), _row_stride(scales)
        self._device = data.get_device()
        self._struct = Rows8Struct(*self._fields)
        self._at = ctypes.addressof(self._struct)

    data = property(lambda self: self._data)
    scales = property(lambda self: self._scales)


def _row_stride(t):
    """Elements between the rows of a 2-D tensor with contiguous rows (one row: its length)."""
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError("rows x channels with contiguous channels expected")
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


# The entry points below are called for steps of a few microseconds: what they
# check costs as little as it can.  OUT_F16 and OUT_F32 by torch's types.
_OUT_TYPES = {}


def _out_type(dtype):
    if dtype in _OUT_TYPES:
        return _OUT_TYPES[dtype]
    import torch

    _OUT_TYPES.update({torch.float16: OUT_F16, torch.float32: OUT_F32})
    if dtype not in _OUT_TYPES:
        raise ValueError(f"f16 or f32 expected, not {dtype}")
    return _OUT_TYPES[dtype]


def _rows_of(ctx, t):
    """(rows, columns, address, type, stride) of a tensor of rows on the context's GPU."""
    shape, strides = t.shape, t.stride()
    if len(shape) != 2 or (strides[1] != 1 and shape[1] > 1):
        raise ValueError("rows x channels with contiguous channels expected")
    rows, c = shape
    stride = strides[0]
    if not t.is_cuda:
        raise ValueError(f"a tensor on the GPU expected, not on {t.device}")
    if t.get_device() != ctx.device:
        raise _elsewhere(ctx, t.device)
    return rows, c, t.data_ptr(), _out_type(t.dtype), stride if rows > 1 or stride > c else c


def _elsewhere(ctx, device):
    return ValueError(f"a tensor on the context's GPU {ctx.device} expected, not on {device}")


def quantize8(ctx, x, out):
    """Rows x k (f16 or f32 tensor) into the Rows8 `out`."""
    rows, k, at, kind, stride = _rows_of(ctx, x)
    if rows != out.rows or k != out.k:
        raise ValueError(f"{tuple(x.shape)} into {out.rows} rows of {out.k}")
    if out._device != ctx.device:
        raise _elsewhere(ctx, out.data.device)
    status = (_lib or load()).ien_quantize8(ctx.h, at, kind, rows, k, stride, out._at)
    if status:
        check(status)


def dequantize8(ctx, x, y):
    """The values of the Rows8 `x` into the rows x k tensor y (f16 or f32)."""
    rows, k, at, kind, stride = _rows_of(ctx, y)
    if rows != x.rows or k != x.k:
        raise ValueError(f"{x.rows} rows of {x.k} into {tuple(y.shape)}")
    if x._device != ctx.device:
        raise _elsewhere(ctx, x.data.device)
    status = (_lib or load()).ien_dequantize8(ctx.h, x._at, rows, k, at, kind, stride)
    if status:
        check(status)


class Matrix8:
    """ien_matrix8: host weights (taps c) x n (numpy f32 or f16) + bias in 8 bits."""

    def __init__(self, ctx, w, bias=None, taps=1):
        import numpy as np

        w = np.ascontiguousarray(w)
        wtype = W_F16 if w.dtype == np.float16 else W_F32
        if wtype == W_F32:
            w = np.ascontiguousarray(w, dtype=np.float32)
        k, n = w.shape
        if k % taps:
            raise ValueError(f"{k} rows of weights in {taps} taps")
        b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float32)
        if b is not None and b.shape != (n,):
            raise ValueError(f"{b.shape} biases for {n} outputs")
        h = ctypes.c_void_p()
        check(load().ien_matrix8_new(ctx.h, _np_ptr(w), wtype, taps, k // taps, n, None if b is None else _np_ptr(b),
                                     ctypes.byref(h)))
        self.h, self.taps, self.c, self.n, self.ctx = h, taps, k // taps, n, ctx

    def free(self):
        if self.h:
            load().ien_matrix8_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


# ien_input8 and ien_output as bytes.
_INPUT8, _OUTPUT = struct.Struct("@iPNPNNNNNi").pack, struct.Struct("@PNii").pack


def _multiply8(ctx, x, shape, row0, matrix, out, act, add, exact):
    rows, n, at, kind, stride = _rows_of(ctx, out)
    if x.k != matrix.c or n != matrix.n:
        raise ValueError(f"rows of {x.k} by {matrix.c} x {matrix.n} into {tuple(out.shape)}")
    if x._device != ctx.device:
        raise _elsewhere(ctx, x.data.device)
    if matrix.ctx.device != ctx.device:
        raise _elsewhere(ctx, f"GPU {matrix.ctx.device}")
    add_at = None
    add_stride = 0
    if add is not None:
        add_rows, add_n, add_at, add_kind, add_stride = _rows_of(ctx, add)
        if add_rows != rows or add_n != n or add_kind != kind:
            raise ValueError("what is added has the output's shape and type")
    status = (_lib or load()).ien_multiply8(ctx.h, _INPUT8(shape[0], *x._fields, *shape[1:], 0 if exact else 1), row0, rows, matrix.h,
                                            _OUTPUT(at, stride, NHWC, kind), act, add_at, add_stride)
    if status:
        check(status)


def multiply8(ctx, x, matrix, out, act=ACT_NONE, add=None, row0=0, exact=True):
    """out = act(x . w + bias + add): rows row0 .. of the Rows8 x, as many as
    out (rows x n, f16 or f32) has; `add` like out, or out itself.  exact=False:
    f16 outputs from the coarser sums of the 8-bit matrix instructions, at twice
    the rate (ien_input8's `fast`); f32 outputs are exact either way."""
    if row0 < 0 or row0 + out.shape[0] > x.rows:
        raise ValueError(f"rows {row0} .. {row0 + out.shape[0]} of {x.rows}")
    _multiply8(ctx, x, (INPUT_ROWS, 1, 1, x.rows, 1), row0, matrix, out, act, add, exact)


def conv8(ctx, x, images, height, width, matrix, out, step=1, act=ACT_NONE, add=None, row0=0, exact=True):
    """The same for a 3 x 3 (9 taps) or 1 x 1 convolution of `images` maps of
    height x width pixels in 8 bits, zero padding: output pixels row0 .., as
    many as out has rows."""
    if images * height * width != x.rows or images < 0 or height < 0 or width < 0 or row0 < 0 or step not in (1, 2):
        raise ValueError(f"{images} maps of {height} x {width} in {x.rows} rows, step {step}, from row {row0}")
    _multiply8(ctx, x, (INPUT_IMAGE, images, height, width, step), row0, matrix, out, act, add, exact)


def _channels_of(ctx, t, c, what="gamma and beta"):
    """The address of c f32 values on the context's GPU, or None."""
    if t is None:
        return None
    if t.shape != (c,) or not t.is_cuda or not t.is_contiguous() or _out_type(t.dtype) != OUT_F32:
        raise ValueError(f"{what} are {c} contiguous f32 values on the GPU")
    if t.get_device() != ctx.device:
        raise _elsewhere(ctx, t.device)
    return t.data_ptr()


def group_norm(ctx, x, images, groups, gamma, beta, y, eps=1e-5, act=ACT_NONE):
    """act(group norm) of `images` maps of x.shape[0] / images pixels (x: rows x
    channels, f16 or f32) into y: a tensor of x's shape (f16 or f32, x itself
    too), or a Rows8.  gamma, beta: f32 tensors, or None for 1 and 0."""
    rows, c, at, kind, stride = _rows_of(ctx, x)
    if images < 1 or rows % images:
        raise ValueError(f"{rows} pixels in {images} maps")
    if isinstance(y, Rows8):
        if y.rows != rows or y.k != c:
            raise ValueError("the result has the input's rows and channels")
        if y._device != ctx.device:
            raise _elsewhere(ctx, y.data.device)
        status = (_lib or load()).ien_group_norm8(
            ctx.h, at, kind, images, rows // images, c, stride, groups, _channels_of(ctx, gamma, c),
            _channels_of(ctx, beta, c), eps, act, y._at)
    else:
        y_rows, y_c, y_at, y_kind, y_stride = _rows_of(ctx, y)
        if y_rows != rows or y_c != c:
            raise ValueError("the result has the input's rows and channels")
        status = (_lib or load()).ien_group_norm(
            ctx.h, at, kind, images, rows // images, c, stride, groups, _channels_of(ctx, gamma, c),
            _channels_of(ctx, beta, c), eps, act, y_at, y_kind, y_stride)
    if status:
        check(status)


def rms_norm(ctx, x, gamma, y=None, rows8=None, add=None, total=None, eps=1e-6):
    """The sum of the rows x and `add` (rows x channels, f16 or f32 each) into
    `total` (x's type; x or add itself too), and its root-mean-square norm times
    gamma (f32 tensor, or None for 1) into y (f16 or f32) and the Rows8 rows8;
    add, total, y and rows8 may each be None."""
    rows, c, at, kind, stride = _rows_of(ctx, x)
    add_at = total_at = y_at = out = None
    add_kind = y_kind = add_stride = total_stride = y_stride = 0
    if add is not None:
        n, k, add_at, add_kind, add_stride = _rows_of(ctx, add)
        if n != rows or k != c:
            raise ValueError("what is added has the input's rows and channels")
    if total is not None:
        n, k, total_at, total_kind, total_stride = _rows_of(ctx, total)
        if n != rows or k != c or total_kind != kind:
            raise ValueError("the sum has the input's rows, channels and type")
    if y is not None:
        n, k, y_at, y_kind, y_stride = _rows_of(ctx, y)
        if n != rows or k != c:
            raise ValueError("the result has the input's rows and channels")
    if rows8 is not None:
        if rows8.rows != rows or rows8.k != c:
            raise ValueError("the result has the input's rows and channels")
        if rows8._device != ctx.device:
            raise _elsewhere(ctx, rows8.data.device)
        out = rows8._at
    status = (_lib or load()).ien_rms_norm(ctx.h, at, kind, rows, c, stride, add_at, add_kind, add_stride, total_at,
                                           total_stride, _channels_of(ctx, gamma, c), eps, y_at, y_kind, y_stride, out)
    if status:
        check(status)


class Routes:
    """ien_routes: each token's experts, best first (`index`: int32, tokens x
    top, -1 for none) and their weights (f32), and the plan that the experts'
    products go by.  The tensors are made here, or given; the plan is route's or
    plan_routes' to fill, again whenever the index changes.  `offsets`: the
    first pair (token x top + slot) of each expert in `order`, which holds the
    pairs in the order of their experts."""

    def __init__(self, tokens, experts, top, index=None, weight=None, device="cuda"):
        import torch

        L = load()
        ints = L.ien_routes_ints(tokens, experts, top)
        if not ints:
            raise ValueError(f"{tokens} tokens with {top} of {experts} experts")
        if index is not None or weight is not None:
            device = (index if index is not None else weight).device
        if index is None:
            index = torch.empty(tokens, top, dtype=torch.int32, device=device)
        if weight is None:
            weight = torch.empty(tokens, top, dtype=torch.float32, device=device)
        for t, dtype in ((index, torch.int32), (weight, torch.float32)):
            if t.shape != (tokens, top) or t.dtype != dtype or not t.is_contiguous() or t.device != index.device:
                raise ValueError(f"the experts and weights are contiguous int32 and f32 tensors of {tokens} x {top} on one device")
        plan = torch.zeros(ints, dtype=torch.int32, device=index.device)  # (zeros: a plan of no pairs)
        if plan.is_cuda:
            torch.cuda.current_stream(plan.device).synchronize()  # (whatever stream the context runs on)
        self.tokens, self.experts, self.top = tokens, experts, top
        self._index, self._weight, self._plan = index, weight, plan
        first = L.ien_routes_order(experts)
        self.offsets, self.order = plan[:experts + 1], plan[first:first + tokens * top]
        self._device = index.get_device()
        self._struct = RoutesStruct(tokens, experts, top, index.data_ptr(), weight.data_ptr(), plan.data_ptr())
        self._at = ctypes.addressof(self._struct)

    index = property(lambda self: self._index)
    weight = property(lambda self: self._weight)


def plan_routes(ctx, routes):
    """The plan of the experts in routes.index (values outside 0 .. experts - 1: none)."""
    if routes._device != ctx.device:
        raise _elsewhere(ctx, routes.index.device)
    check((_lib or load()).ien_routes_plan(ctx.h, routes._at))


# ien_router as bytes.
_ROUTER = struct.Struct("@iPNNNif").pack


def route(ctx, logits, routes, score=SCORE_SOFTMAX, bias=None, groups=1, kept=None, group_top=1, renormalise=True, scale=1.0):
    """Each token's experts and weights from its logits (tokens x experts, f16
    or f32), and their plan, into `routes`: see ien_router.  kept: all groups by
    default."""
    tokens, experts, at, kind, stride = _rows_of(ctx, logits)
    if tokens != routes.tokens or experts != routes.experts:
        raise ValueError(f"{tuple(logits.shape)} logits for {routes.tokens} tokens of {routes.experts} experts")
    if routes._device != ctx.device:
        raise _elsewhere(ctx, routes.index.device)
    if groups < 1 or group_top < 1 or (kept is not None and kept < 1):
        raise ValueError(f"{kept} of {groups} groups by their {group_top} best")
    how = _ROUTER(score, _channels_of(ctx, bias, experts, "biases") or 0, groups, groups if kept is None else kept, group_top,
                  1 if renormalise else 0, scale)
    status = (_lib or load()).ien_route(ctx.h, at, kind, stride, how, routes._at)
    if status:
        check(status)


class Experts8:
    """ien_experts8: experts x c x n weights (f32 or f16; torch on the context's
    GPU, or numpy) and experts x n biases in 8 bits.  gated: n / 2 outputs, the
    activation of the first half of the columns times the second half."""

    def __init__(self, ctx, w, bias=None, gated=False):
        import torch

        device = torch.device("cuda", ctx.device)

        def held(t, types):
            t = t if isinstance(t, torch.Tensor) else torch.from_numpy(t)
            if t.is_cuda and t.get_device() != ctx.device:
                raise _elsewhere(ctx, t.device)
            return t.to(device, t.dtype if t.dtype in types else torch.float32).contiguous()

        if len(w.shape) != 3 or (bias is not None and tuple(bias.shape) != (w.shape[0], w.shape[2])):
            raise ValueError("weights are experts x c x n, biases experts x n")
        w = held(w, (torch.float16, torch.float32))
        b = None if bias is None else held(bias, (torch.float32,))
        torch.cuda.current_stream(device).synchronize()  # (they may have been made on another stream than the context's)
        experts, c, n = w.shape
        h = ctypes.c_void_p()
        check(load().ien_experts8_new(ctx.h, _ptr(w), W_F16 if w.dtype == torch.float16 else W_F32, experts, c, n,
                                      1 if gated else 0, _ptr(b), ctypes.byref(h)))
        self.h, self.experts, self.c, self.n, self.gated, self.ctx = h, experts, c, n // 2 if gated else n, gated, ctx

    def free(self):
        if self.h:
            load().ien_experts8_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def _experts_of(ctx, rows8, rows, routes, matrix):
    if rows8.k != matrix.c or rows8.rows != rows or routes.experts != matrix.experts:
        raise ValueError(f"{rows8.rows} rows of {rows8.k} by {matrix.experts} experts of {matrix.c} x {matrix.n}, routes of "
                         f"{routes.tokens} tokens to {routes.top} of {routes.experts}")
    if rows8._device != ctx.device:
        raise _elsewhere(ctx, rows8.data.device)
    if routes._device != ctx.device:
        raise _elsewhere(ctx, routes.index.device)
    if matrix.ctx.device != ctx.device:
        raise _elsewhere(ctx, f"GPU {matrix.ctx.device}")


def experts_in8(ctx, x, routes, matrix, out, act=ACT_NONE, exact=True):
    """The Rows8 out (tokens x top rows, in the order of routes.order) from the
    Rows8 x (a row a token): act(x . w + bias) of each pair's expert, of gated
    weights act(gate) x up.  exact=False: the coarser sums of multiply8."""
    _experts_of(ctx, x, routes.tokens, routes, matrix)
    if out.rows != routes.tokens * routes.top or out.k != matrix.n:
        raise ValueError(f"{routes.tokens} x {routes.top} rows of {matrix.n} into {out.rows} of {out.k}")
    if out._device != ctx.device:
        raise _elsewhere(ctx, out.data.device)
    status = (_lib or load()).ien_experts_in8(ctx.h, x._at, routes._at, matrix.h, act, 0 if exact else 1, out._at)
    if status:
        check(status)


def expert_parts(routes, matrix, dtype):
    """What experts_out8 writes its products to: of the result's type, or f32."""
    import torch

    return torch.empty(load().ien_experts_parts(routes._at, matrix.h), dtype=dtype, device=routes.index.device)


def experts_out8(ctx, h, routes, matrix, parts, out, add=None, exact=True, branch=None):
    """out (tokens x n, f16 or f32) = (add + branch) + each token's sum of weight x
    (h . w + bias) over its pairs' rows of the Rows8 h (as experts_in8 leaves
    them); `add` like out, or out itself; `branch` f16 or f32, or out itself;
    parts: expert_parts(routes, matrix, out's type or f32).  Products are rounded
    to the parts' type (in f16 those past 65504 are infinite), sums are in f32."""
    _experts_of(ctx, h, routes.tokens * routes.top, routes, matrix)
    rows, n, at, kind, stride = _rows_of(ctx, out)
    if rows != routes.tokens or n != matrix.n:
        raise ValueError(f"{routes.tokens} rows of {matrix.n} into {tuple(out.shape)}")
    if not parts.is_contiguous() or parts.get_device() != ctx.device or parts.numel() < rows * routes.top * (-(-n // 8) * 8) \
            or _out_type(parts.dtype) not in (kind, OUT_F32):
        raise ValueError("parts are what expert_parts makes for the result's type or f32")
    add_at = branch_at = None
    add_stride = branch_stride = 0
    branch_kind = kind
    if add is not None:
        add_rows, add_n, add_at, add_kind, add_stride = _rows_of(ctx, add)
        if add_rows != rows or add_n != n or add_kind != kind:
            raise ValueError("what is added has the output's shape and type")
    if branch is not None:
        add_rows, add_n, branch_at, branch_kind, branch_stride = _rows_of(ctx, branch)
        if add_rows != rows or add_n != n:
            raise ValueError("the branch has the output's shape")
    status = (_lib or load()).ien_experts_out8_ex(ctx.h, h._at, routes._at, matrix.h, 0 if exact else 1, parts.data_ptr(),
                                                  _out_type(parts.dtype), add_at, add_stride, branch_at, branch_kind,
                                                  branch_stride, _OUTPUT(at, stride, NHWC, kind))
    if status:
        check(status)


def bytes_to_floats(ctx, src, dst):
    """to_float on device: uint8 tensor to float32 tensor of the same size."""
    check(load().ien_bytes_to_floats(ctx.h, _ptr(src), _ptr(dst), src.numel()))


def floats_to_bytes(ctx, src, dst):
    """to_byte on device: float32 tensor to uint8 tensor of the same size."""
    check(load().ien_floats_to_bytes(ctx.h, _ptr(src), _ptr(dst), src.numel()))


def mask_bytes(ctx, mask, dst):
    check(load().ien_mask_bytes(ctx.h, _ptr(mask), _ptr(dst), mask.numel()))


def normalize_bytes(ctx, rgb, mean, std, dst):
    """rgb: uint8 tensor of pixels x 3 values; mean, std: three floats."""
    m = (ctypes.c_float * 3)(*mean)
    d = (ctypes.c_float * 3)(*std)
    check(load().ien_normalize_bytes(ctx.h, _ptr(rgb), rgb.numel() // 3, m, d, _ptr(dst)))


def composite_bytes(ctx, rgb, mask, pred, out):
    check(load().ien_composite_bytes(ctx.h, _ptr(rgb), _ptr(mask), _ptr(pred), mask.numel(), _ptr(out)))


class Model:
    """ien_model: the reference's Model with the HIP engine."""

    def __init__(self, ctx, kind, tensors=None, path=None):
        import numpy as np

        self.kind = kind
        L = load()
        h = ctypes.c_void_p()
        if path is not None:
            check(L.ien_model_load(ctx.h, kind, str(path).encode(), ctypes.byref(h)))
        else:
            arr = (Tensor * len(tensors))()
            keep = []
            for j, (name, value) in enumerate(tensors.items()):
                v = np.ascontiguousarray(value, dtype=np.float32)
                keep.append(v)
                arr[j].name = name.encode()
                arr[j].rank = v.ndim
                for d, s in enumerate(v.shape):
                    arr[j].dims[d] = s
                arr[j].values = v.ctypes.data
            check(L.ien_model_from_tensors(ctx.h, kind, arr, len(tensors), ctypes.byref(h)))
        self.h, self.ctx = h, ctx

    def free(self):
        if self.h:
            load().ien_model_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def set_graph(self, enabled):
        check(load().ien_model_set_graph(self.h, int(enabled)))

    def run(self, image, progress=None, mask=None):
        """Host f32 H x W x 3 in, host f32 out (Model::run_float): 4H x 4W x 3
        for Real-ESRGAN, H x W x 3 for SCUNet and LaMa (which takes the
        H x W mask, 1 = fill), H x W logits for BiRefNet (whose input is
        already normalised)."""
        import numpy as np

        image = np.ascontiguousarray(image, dtype=np.float32)
        h, w, _ = image.shape
        s = 4 if self.kind == MODEL_REALESRGAN else 1
        shape = (h, w) if self.kind == MODEL_BIREFNET else (s * h, s * w, 3)
        out = np.empty(shape, np.float32)
        m = None if mask is None else np.ascontiguousarray(mask, dtype=np.float32)
        cb = PROGRESS(progress) if progress else None
        check(load().ien_model_run(self.h, image.ctypes.data_as(ctypes.c_void_p),
                                   None if m is None else m.ctypes.data_as(ctypes.c_void_p), w, h,
                                   out.ctypes.data_as(ctypes.c_void_p),
                                   ctypes.cast(cb, ctypes.c_void_p) if cb else None, None))
        return out

    def run_tiled(self, image, tile, margin, progress=None):
        """Model::run_float_tiled (Real-ESRGAN, SCUNet): host f32 H x W x 3
        in, the run's output shape out."""
        import numpy as np

        image = np.ascontiguousarray(image, dtype=np.float32)
        h, w, _ = image.shape
        s = 4 if self.kind == MODEL_REALESRGAN else 1
        out = np.empty((s * h, s * w, 3), np.float32)
        cb = PROGRESS(progress) if progress else None
        check(load().ien_model_run_tiled(self.h, image.ctypes.data_as(ctypes.c_void_p), w, h, tile, margin,
                                         out.ctypes.data_as(ctypes.c_void_p),
                                         ctypes.cast(cb, ctypes.c_void_p) if cb else None, None))
        return out

    def run_u8(self, rgb, mask=None, progress=None):
        """Model::run on 8-bit RGB H x W x 3 (uint8): bytes out (4H x 4W x 3
        for Real-ESRGAN, H x W x 3 for SCUNet and LaMa, which takes the
        H x W byte mask), H x W f32 logits for BiRefNet."""
        import numpy as np

        rgb = np.ascontiguousarray(rgb, dtype=np.uint8)
        h, w, _ = rgb.shape
        if self.kind == MODEL_BIREFNET:
            out = np.empty((h, w), np.float32)
        else:
            s = 4 if self.kind == MODEL_REALESRGAN else 1
            out = np.empty((s * h, s * w, 3), np.uint8)
        m = None if mask is None else np.ascontiguousarray(mask, dtype=np.uint8)
        cb = PROGRESS(progress) if progress else None
        check(load().ien_model_run_u8(self.h, rgb.ctypes.data_as(ctypes.c_void_p),
                                      None if m is None else m.ctypes.data_as(ctypes.c_void_p), w, h,
                                      out.ctypes.data_as(ctypes.c_void_p),
                                      ctypes.cast(cb, ctypes.c_void_p) if cb else None, None))
        return out

    def run_device(self, d_image, width, height, d_out, d_mask=None):
        check(load().ien_model_run_device(self.h, _ptr(d_image), None if d_mask is None else _ptr(d_mask),
                                          width, height, _ptr(d_out)))

    def status(self):
        """Waits for the model's stream; raises IenError (ERR_GPU) when a chain
        launched by run_device since the last report gave up."""
        check(load().ien_model_status(self.h))
