"""ctypes binding of libdsv4_b200.so (include/dsv4_b200.h).

The product's Python face: the same C ABI the reference's C host links
against, reachable from numpy (host buffers, layer 1) and from torch CUDA
tensors (device pointers, layer 2). There is no CPU fallback: loading fails
loudly when the library is missing, and every call that the C ABI rejects
raises.
"""
import ctypes as C
import os
import subprocess

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libdsv4_b200.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "dsv4_b200.h")

WF32, WBF16, WFP8, WFP4 = 0, 1, 2, 3


class QMat(C.Structure):
    """The reference's DSV4QMat (include/dsv4/dsv4.h:208-214)."""
    _fields_ = [("w", C.c_void_p), ("s", C.c_void_p), ("wdt", C.c_int),
                ("rows", C.c_int), ("cols", C.c_int),
                ("blk_r", C.c_int), ("blk_c", C.c_int)]


ROPE_MAX = 256                  # DSV4B_ROPE_MAX: rotated elements of a head
KVQ_MAX_D = 576                 # DSV4B_KVQ_MAX_D: elements of a cache row
TREE_MAX = 64                   # DSV4B_TREE_MAX: drafted tokens of a sequence
ROPE_INTERLEAVED, ROPE_HALF = 0, 1


class RopeCfg(C.Structure):
    """dsv4b_rope_cfg: angle per position of every pair, and the layout."""
    _fields_ = [("freq", C.c_double * (ROPE_MAX // 2)), ("rd", C.c_int), ("layout", C.c_int)]


class KvqC(C.Structure):
    """dsv4b_kvq."""
    _fields_ = [("codes", C.c_void_p), ("scales", C.c_void_p), ("n_pages", C.c_long),
                ("page_rows", C.c_int), ("d", C.c_int), ("tail", C.c_int)]


class LogitAdjustC(C.Structure):
    """dsv4b_logit_adjust."""
    _fields_ = [("hist", C.c_void_p), ("hist_stride", C.c_long), ("hist_len", C.c_void_p), ("n_prompt", C.c_void_p),
                ("rep", C.c_void_p), ("freq", C.c_void_p), ("pres", C.c_void_p), ("bias_ids", C.c_void_p),
                ("bias", C.c_void_p), ("bias_stride", C.c_long), ("bias_len", C.c_void_p), ("mask", C.c_void_p),
                ("mask_stride", C.c_long)]


def build():
    """Compile the library in-tree (nvcc cross-compiles without a GPU)."""
    subprocess.run(["make", "-C", HERE, "-j8"], check=True)
    return LIB_PATH


_lib = None


def lib():
    """Load libdsv4_b200.so once; raise if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError("libdsv4_b200.so is not built (run `make -C %s`)" % HERE)
        _lib = C.CDLL(LIB_PATH)
        _declare(_lib)
    return _lib


def _declare(L):
    vp, i, f, sz = C.c_void_p, C.c_int, C.c_float, C.c_size_t
    qp = C.POINTER(QMat)
    sig = {
        "dsv4_cuda_available": ([], i),
        "dsv4_cuda_init": ([], i),
        "dsv4_cuda_set_blocking_sync": ([], i),
        "dsv4_cuda_upload": ([qp], i),
        "dsv4_cuda_has": ([qp], i),
        "dsv4_cuda_mmq": ([vp, vp, qp], None),
        "dsv4_cuda_mmq_n": ([vp, vp, qp, i], None),
        "dsv4_cuda_free_vram": ([], sz),
        "dsv4_cuda_shutdown": ([], None),
        "dsv4_cuda_dump_e4m3": ([vp], i),
        "dsv4_cuda_evict": ([qp], i),
        "dsv4_cuda_resident_ptrs": ([qp, C.POINTER(vp), C.POINTER(vp)], i),
        "dsv4b_gemv": ([i, vp, vp, vp, vp, i, i, i, i, i, vp], i),
        "dsv4_cuda_moe_prepare": ([qp, vp, qp, i, qp, i, f, i, f], vp),
        "dsv4_cuda_moe": ([vp, vp, vp, vp, vp, vp], i),
        "dsv4_cuda_moe_free": ([vp], None),
        "dsv4b_moe_forward": ([vp, vp, vp, vp], i),
        "dsv4_cuda_indexer_score": ([vp, vp, vp, vp, i, i, i], i),
        "dsv4_cuda_topk": ([vp, vp, i, i], i),
        "dsv4_cuda_sparse_attn": ([vp, vp, vp, vp, vp, i, i, i, f], i),
        "dsv4b_indexer_score": ([vp, vp, vp, i, C.c_long, C.c_long, vp, i, i, i, f, i, vp], i),
        "dsv4b_topk": ([vp, vp, i, i, i, vp], i),
        "dsv4b_sparse_attn_scratch": ([i, i, i, i], sz),
        "dsv4b_sparse_attn": ([vp, vp, vp, i, C.c_long, vp, vp, i, i, i, f, i, vp, sz, vp], i),
        "dsv4b_rope_init": ([C.POINTER(RopeCfg), i, i, C.c_double, C.c_double, i, C.c_double, C.c_double], i),
        "dsv4b_rope": ([vp, i, C.c_long, C.c_long, vp, i, C.c_long, C.c_long, vp, vp, i, i, i, i, i, vp], i),
        "dsv4b_kv_write": ([vp, vp, i, C.c_long, vp, i, vp, vp, vp], i),
        "dsv4b_kv_read": ([vp, vp, i, C.c_long, vp, i, vp], i),
        "dsv4b_tree_attn_scratch": ([i, i, i, i, i], sz),
        "dsv4b_tree_attn": ([vp, vp, i, C.c_long, C.c_long, vp, vp, i, vp, vp, vp, vp, i, i, i, i, f, vp, sz, vp], i),
        "dsv4b_tree_attn_status": ([], i),
        "dsv4b_tree_attn_selftest": ([i, vp], i),
        "dsv4b_logits": ([vp, vp, i, C.c_long, C.c_long, vp, vp, i, i, vp], i),
        "dsv4_cuda_model_create": ([vp, vp, vp, vp, i], vp),
        "dsv4_cuda_model_begin": ([vp, vp, i], i),
        "dsv4_cuda_model_step": ([vp, vp, vp], i),
        "dsv4_cuda_model_generate": ([vp, vp, i, i, vp], i),
        "dsv4_cuda_model_free": ([vp], None),
        "dsv4b_model_step_async": ([vp, vp], i),
        "dsv4_cuda_model_decode": ([vp, i, i, vp], i),
        "dsv4_cuda_model_create_synthetic": ([vp, i, C.c_ulonglong], vp),
        "dsv4_cuda_model_create_synthetic_batch": ([vp, i, C.c_ulonglong, i], vp),
        "dsv4_cuda_model_create_batch": ([vp, vp, vp, vp, i, i], vp),
        "dsv4b_model_n_seq": ([vp], i),
        "dsv4b_model_begin_batch": ([vp, vp, i], i),
        "dsv4b_model_generate_batch": ([vp, vp, i, i, vp], i),
        "dsv4b_model_decode_batch": ([vp, vp, i, vp], i),
        "dsv4b_model_prefill": ([vp, vp, i, i], i),
        "dsv4b_model_generate_prefill": ([vp, vp, i, i, i, vp], i),
        "dsv4b_model_prefill_kernels": ([vp], i),
        "dsv4b_model_stream": ([vp], vp),
        "dsv4_cuda_model_bytes": ([vp], sz),
        "dsv4_cuda_model_step_kernels": ([vp], i),
        "dsv4b_shard_check": ([vp, i], i),
        "dsv4b_shard_plan": ([vp, i, i, vp], i),
        "dsv4b_model_comm_status": ([vp], i),
        "dsv4b_nccl_id_bytes": ([], sz),
        "dsv4b_nccl_unique_id": ([vp], i),
        "dsv4_cuda_model_create_synthetic_sharded": ([vp, i, C.c_ulonglong, i, i, vp], vp),
    }
    for name, (args, res) in sig.items():
        fn = getattr(L, name)
        fn.argtypes, fn.restype = args, res


def header_functions():
    """Names of every function include/dsv4_b200.h declares."""
    import re
    txt = open(HEADER).read()
    txt = re.sub(r"/\*.*?\*/", "", txt, flags=re.S)
    return sorted(set(re.findall(r"\b(dsv4b?_\w+)\s*\(", txt)))


def check(rc, what):
    if rc != 0:
        raise RuntimeError("%s failed (rc=%d)" % (what, rc))


def ptr(a):
    """Address of a numpy array or torch tensor."""
    if isinstance(a, np.ndarray):
        return a.ctypes.data
    return a.data_ptr()


def stream_ptr(s=None):
    return None if s is None else s.cuda_stream


# ----------------------------------------------------------- host-side API

class Matrix:
    """A host matrix in one of the checkpoint formats, kept alive while it is
    resident (the backend keys residency on the host pointer, as the
    reference's does)."""

    def __init__(self, wdt, W, S=None, rows=None, cols=None, blk=None):
        self.W = np.ascontiguousarray(W)
        self.S = None if S is None else np.ascontiguousarray(S, dtype=np.uint8)
        if rows is None:
            rows = self.W.shape[0]
        if cols is None:
            cols = {WF32: self.W.shape[1], WBF16: self.W.shape[1],
                    WFP8: self.W.shape[1], WFP4: self.W.shape[1] * 2}[wdt]
        if blk is None:
            blk = {WFP8: (128, 128), WFP4: (1, 32)}.get(wdt, (0, 0))
        self.q = QMat(self.W.ctypes.data, None if self.S is None else self.S.ctypes.data,
                      wdt, rows, cols, blk[0], blk[1])

    def slice_rows(self, r0, nrows):
        """A DSV4QMat of rows [r0, r0+nrows), sharing this matrix's bytes --
        the way the reference layer slices wo_a per group."""
        m = Matrix.__new__(Matrix)
        m.W, m.S = self.W, self.S
        q = self.q
        rb = {WF32: 4 * q.cols, WBF16: 2 * q.cols, WFP8: q.cols, WFP4: q.cols // 2}[q.wdt]
        s = None
        if self.S is not None:
            sc = -(-q.cols // q.blk_c)
            s = self.S.ctypes.data + (r0 // q.blk_r) * sc
        m.q = QMat(self.W.ctypes.data + r0 * rb, s, q.wdt, nrows, q.cols, q.blk_r, q.blk_c)
        return m

    def upload(self):
        rc = lib().dsv4_cuda_upload(C.byref(self.q))
        self._owned = (rc == 0)
        return rc

    def evict(self):
        if getattr(self, "_owned", False):
            self._owned = False
            return lib().dsv4_cuda_evict(C.byref(self.q))
        return -1

    def __del__(self):
        # Residency is keyed on the host address (as in the reference); once
        # this buffer is freed the address may be reused by another matrix.
        try:
            self.evict()
        except Exception:
            pass

    def has(self):
        return lib().dsv4_cuda_has(C.byref(self.q))

    def mmq(self, x):
        x = np.ascontiguousarray(x, np.float32)
        nt = x.size // self.q.cols
        y = np.empty(nt * self.q.rows, np.float32)
        if nt == 1:
            lib().dsv4_cuda_mmq(y.ctypes.data, x.ctypes.data, C.byref(self.q))
        else:
            lib().dsv4_cuda_mmq_n(y.ctypes.data, x.ctypes.data, C.byref(self.q), nt)
        return y.reshape(nt, self.q.rows) if nt > 1 else y

    def device_ptrs(self):
        dw, ds = C.c_void_p(), C.c_void_p()
        check(lib().dsv4_cuda_resident_ptrs(C.byref(self.q), C.byref(dw), C.byref(ds)),
              "dsv4_cuda_resident_ptrs")
        return dw.value, ds.value


def init():
    L = lib()
    if not L.dsv4_cuda_available():
        raise RuntimeError("no CUDA device: the B200 backend has no CPU fallback")
    check(L.dsv4_cuda_init(), "dsv4_cuda_init")
    return L


def dump_e4m3():
    out = np.empty(256, np.float32)
    check(lib().dsv4_cuda_dump_e4m3(out.ctypes.data), "dsv4_cuda_dump_e4m3")
    return out


# ---------------------------------------------------------- device-side API

def gemv(wdt, y, x, W, S, rows, cols, blk_r=0, blk_c=0, nt=1, stream=None):
    check(lib().dsv4b_gemv(wdt, ptr(y), ptr(x), W if isinstance(W, int) else ptr(W),
                           None if S is None else (S if isinstance(S, int) else ptr(S)),
                           rows, cols, blk_r, blk_c, nt, stream_ptr(stream)), "dsv4b_gemv")


class MoE:
    """One layer's MoE bound to resident matrices (dsv4_cuda_moe_prepare)."""

    def __init__(self, gate, experts, shared=None, bias=None, topk=6, route_scale=1.0,
                 score_func=2, swiglu_limit=10.0):
        self.gate, self.experts, self.shared = gate, experts, shared
        n = len(experts)
        self._qs = (QMat * (3 * n))(*[m.q for trio in experts for m in trio])
        self._sh = None if shared is None else (QMat * 3)(*[m.q for m in shared])
        self.bias = None if bias is None else np.ascontiguousarray(bias, np.float32)
        self.topk, self.hidden = topk, gate.q.cols
        self.h = lib().dsv4_cuda_moe_prepare(C.byref(gate.q),
                                             None if self.bias is None else self.bias.ctypes.data,
                                             self._qs, n, self._sh, topk, route_scale, score_func,
                                             swiglu_limit)
        if not self.h:
            raise RuntimeError("dsv4_cuda_moe_prepare failed (matrix not resident or bad shapes)")

    def __call__(self, x, fixed=None):
        x = np.ascontiguousarray(x, np.float32)
        out = np.empty(self.hidden, np.float32)
        idx = np.empty(self.topk, np.int32)
        w = np.empty(self.topk, np.float32)
        fx = None if fixed is None else np.ascontiguousarray(fixed, np.int32)
        check(lib().dsv4_cuda_moe(self.h, out.ctypes.data, x.ctypes.data,
                                  None if fx is None else fx.ctypes.data, idx.ctypes.data,
                                  w.ctypes.data), "dsv4_cuda_moe")
        return out, idx, w

    def forward_dev(self, out, x, stream=None):
        check(lib().dsv4b_moe_forward(self.h, ptr(out), ptr(x), stream_ptr(stream)), "dsv4b_moe_forward")

    def close(self):
        if self.h:
            lib().dsv4_cuda_moe_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ------------------------------------------------------------- sparse MLA

F32, BF16, E4M3 = 0, 1, 2
# DSV4B_SPARSE_ATTN_STATIC_SCRATCH: the fixed device array of dsv4b_sparse_attn_static
SPARSE_ATTN_STATIC_SCRATCH = 8 << 20


def _f(a):
    return np.ascontiguousarray(a, np.float32)


def indexer_score(q, kv, weights):
    """dsv4_cuda_indexer_score: reference signature, host buffers."""
    q, kv, w = _f(q), _f(kv), _f(weights)
    n_heads, head_dim = q.shape
    out = np.empty(kv.shape[0], np.float32)
    check(lib().dsv4_cuda_indexer_score(out.ctypes.data, q.ctypes.data, kv.ctypes.data, w.ctypes.data,
                                        n_heads, head_dim, kv.shape[0]), "dsv4_cuda_indexer_score")
    return out


def topk(scores, k):
    scores = _f(scores)
    idx = np.empty(max(1, min(k, scores.size)), np.int32)
    n = lib().dsv4_cuda_topk(idx.ctypes.data, scores.ctypes.data, scores.size, k)
    if n < 0:
        raise RuntimeError("dsv4_cuda_topk failed")
    return idx[:n]


def sparse_attn(q, kv, sink, idxs, scale):
    q, kv, sink = _f(q), _f(kv), _f(sink)
    idxs = np.ascontiguousarray(idxs, np.int32)
    h, d = q.shape
    o = np.empty((h, d), np.float32)
    check(lib().dsv4_cuda_sparse_attn(o.ctypes.data, q.ctypes.data, kv.ctypes.data, sink.ctypes.data,
                                      idxs.ctypes.data, h, d, idxs.size, scale), "dsv4_cuda_sparse_attn")
    return o


def indexer_score_dev(out, q, keys, key_dt, key_stride, seq_key_stride, w, n_heads, head_dim, n_pos,
                      scale, batch, stream=None):
    check(lib().dsv4b_indexer_score(ptr(out), ptr(q), ptr(keys), key_dt, key_stride, seq_key_stride,
                                    ptr(w), n_heads, head_dim, n_pos, scale, batch, stream_ptr(stream)),
          "dsv4b_indexer_score")


def topk_dev(idx, scores, n, k, batch, stream=None):
    check(lib().dsv4b_topk(ptr(idx), ptr(scores), n, k, batch, stream_ptr(stream)), "dsv4b_topk")


def sparse_attn_scratch(n_heads, d, topk_n, batch):
    return lib().dsv4b_sparse_attn_scratch(n_heads, d, topk_n, batch)


def sparse_attn_dev(o, q, kv, kv_dt, seq_kv_rows, sink, idxs, n_heads, d, topk_n, scale, batch,
                    scratch, stream=None):
    nbytes = scratch.numel() * scratch.element_size()
    check(lib().dsv4b_sparse_attn(ptr(o), ptr(q), ptr(kv), kv_dt, seq_kv_rows, ptr(sink), ptr(idxs),
                                  n_heads, d, topk_n, scale, batch, ptr(scratch), nbytes,
                                  stream_ptr(stream)), "dsv4b_sparse_attn")


# ----------------------------------------- verifying a tree of drafted tokens
#
# These take torch CUDA tensors of one device and check them (ValueError) before
# the C ABI does. With stream=None they run on torch's current stream of that
# device, so they are ordered after the torch work that made their tensors. With
# another stream the caller orders it (Stream.wait_stream); its tensors' memory is
# not given out again before the call there has ended.

F16 = 3
_t = None                       # torch, imported by the first of these calls
_row_dt = {}


def _torch():
    global _t
    if _t is None:
        import torch
        _row_dt.update({torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16})
        _t = torch
    return _t


def _int(v, what):
    """v as a C int: ctypes would keep its low 32 bits."""
    v = int(v)
    if not -0x80000000 <= v <= 0x7FFFFFFF:
        raise ValueError("%s is out of range" % what)
    return v


def _too_long():
    raise ValueError("a size or an offset is not in 0 .. 2^31 - 1")


def _dt(t, what):
    """The row type (F32, BF16, F16) of a tensor."""
    dt = _row_dt.get(t.dtype)
    if dt is None:
        raise ValueError("%s must be float32, bfloat16 or float16" % what)
    return dt


def _want(t, what, dev, dtype, shape=None):
    """Address of a contiguous tensor on CUDA device `dev` (its index) of the
    given type and shape (None: any)."""
    if t.get_device() != dev:
        raise ValueError("%s must be on the device of the other tensors" % what)
    if t.dtype is not dtype:
        raise ValueError("%s must be %s" % (what, dtype))
    if shape is not None and t.shape != shape:
        raise ValueError("%s must have shape %s" % (what, shape))
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % what)
    return t.data_ptr()


def _stream(dev, stream, tensors):
    """The handle to enqueue on: torch's current stream of the device for None
    (its default stream by the legacy handle, as NULL is the backend's own).
    The tensors of a call on a given stream are recorded there."""
    if stream is None:
        return _t._C._cuda_getCurrentRawStream(dev) or 1
    if stream.device.index != dev:
        raise ValueError("the stream belongs to another device than the tensors")
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
    return stream.cuda_stream or 1


def _enqueue(fn, what, dev, *args):
    """fn(*args) with device dev current."""
    if _t._C._cuda_getDevice() == dev:
        rc = fn(*args)
    else:
        with _t.cuda.device(dev):
            rc = fn(*args)
    if rc != 0:
        raise RuntimeError("%s %s (rc=%d)" % (what, "refused its arguments" if rc == -1 else "could not launch", rc))


def rope_cfg(rd, base, layout=ROPE_INTERLEAVED, factor=1.0, orig=0, beta_fast=32.0, beta_slow=1.0):
    """Frequencies of a rotation of rd elements (dsv4b_rope_init); orig > 0
    scales them by factor for contexts beyond orig positions."""
    r = RopeCfg()
    check(lib().dsv4b_rope_init(C.byref(r), _int(rd, "rd"), _int(layout, "layout"), float(base), float(factor),
                                _int(orig, "orig"), float(beta_fast), float(beta_slow)), "dsv4b_rope_init")
    return r


def rope_dev(out, x, pos, cfg, first, inverse=False, stream=None):
    """out = x [tokens, heads, width] with elements first .. first + cfg.rd of
    every head rotated to pos [tokens] (int32); inverse rotates back. Unit-stride
    heads, else any strides of x, and of out those in which no two heads
    interleave (a transposed [heads, tokens, width] too); out may be x."""
    i32 = _torch().int32
    dev = x.get_device()
    xs, os_, shape = x.stride(), out.stride(), x.shape
    if len(shape) != 3 or out.shape != shape or xs[2] != 1 or os_[2] != 1:
        raise ValueError("x and out must be [tokens, heads, width] with unit-stride heads")
    if dev < 0 or out.get_device() != dev:
        raise ValueError("x and out must be on one CUDA device")
    n, h, w = shape
    first = int(first)
    if (n | h | w | first) >> 31:
        _too_long()
    # torch leaves the stride of a length-1 axis free
    xh, oh = (xs[1], os_[1]) if h > 1 else (w, w)
    xt, ot = (xs[0], os_[0]) if n > 1 else ((h - 1) * xh + w, (h - 1) * oh + w)
    _enqueue(lib().dsv4b_rope, "dsv4b_rope", dev, out.data_ptr(), _dt(out, "out"), ot, oh, x.data_ptr(), _dt(x, "x"),
             xt, xh, C.addressof(cfg), _want(pos, "pos", dev, i32, (n,)), n, h, w, first, 1 if inverse else 0,
             _stream(dev, stream, (out, x, pos)))


class KvCache:
    """A paged cache of quantised rows (dsv4b_kvq) in the caller's tensors:
    codes [pages, page_rows, d + tail] and scales [pages, page_rows], uint8.
    page_rows is a power of two; d and tail are multiples of 64."""

    def __init__(self, codes, scales, d, tail):
        if codes.dim() != 3 or codes.shape[2] != d + tail:
            raise ValueError("codes must be [pages, page_rows, d + tail]")
        pages, rows = codes.shape[:2]
        if d < 64 or d > KVQ_MAX_D or d % 64 or tail < 0 or tail > d or tail % 64:
            raise ValueError("d must be a multiple of 64 up to %d, tail one up to d" % KVQ_MAX_D)
        if rows < 1 or rows & (rows - 1) or pages < 1:
            raise ValueError("page_rows must be a power of two, and there must be a page")
        self.device = codes.get_device()
        if self.device < 0:
            raise ValueError("codes must be on a CUDA device")
        u8 = _torch().uint8
        self.c = KvqC(_want(codes, "codes", self.device, u8), _want(scales, "scales", self.device, u8, (pages, rows)),
                      pages, rows, d, tail)
        self.codes, self.scales, self.d, self.tail = codes, scales, d, tail
        self.ref = C.addressof(self.c)

    @classmethod
    def empty(cls, pages, page_rows, d, tail, device="cuda"):
        """A cache of newly allocated, zeroed pages."""
        import torch
        return cls(torch.zeros((pages, page_rows, d + tail), dtype=torch.uint8, device=device),
                   torch.zeros((pages, page_rows), dtype=torch.uint8, device=device), d, tail)


def _rows(t, what, cache):
    s, n = t.stride(), t.shape
    if len(n) != 2 or n[1] != cache.d or s[1] != 1 or t.get_device() != cache.device:
        raise ValueError("%s must be [n, d] with unit-stride rows on the cache's device" % what)
    if n[0] >> 31:
        _too_long()
    return t.data_ptr(), _dt(t, what), s[0] if n[0] > 1 else cache.d, n[0]


def kv_write_dev(cache, rows, slots, rope=None, pos=None, stream=None):
    """Quantise rows [n, d] into the cache's slots [n] (int64, distinct; -1
    skips a row). With rope and pos [n] (int32) the last rope.rd elements of
    each row are rotated first."""
    p, dt, st, n = _rows(rows, "rows", cache)
    dev = cache.device
    if (rope is None) != (pos is None):
        raise ValueError("rope and pos go together")
    _enqueue(lib().dsv4b_kv_write, "dsv4b_kv_write", dev, cache.ref, p, dt, st,
             _want(slots, "slots", dev, _t.int64, (n,)), n, None if rope is None else C.addressof(rope),
             None if pos is None else _want(pos, "pos", dev, _t.int32, (n,)),
             _stream(dev, stream, (cache.codes, cache.scales, rows, slots, pos)))


def kv_read_dev(out, cache, slots, stream=None):
    """out [n, d] = the values of the cache's rows slots [n]; zeros for a slot
    outside the cache."""
    p, dt, st, n = _rows(out, "out", cache)
    dev = cache.device
    _enqueue(lib().dsv4b_kv_read, "dsv4b_kv_read", dev, cache.ref, p, dt, st,
             _want(slots, "slots", dev, _t.int64, (n,)), n,
             _stream(dev, stream, (out, cache.codes, cache.scales, slots)))


def tree_mask(parents):
    """Ancestor masks (int64, for tree_attn_dev) of drafted tokens: parents[i]
    is the index of token i's parent among the drafted tokens (an earlier one),
    or -1 for a child of the context. Every token attends to itself."""
    m = []
    for i, p in enumerate(parents):
        if i >= TREE_MAX or not -1 <= p < i:
            raise ValueError("at most %d tokens, each after its parent" % TREE_MAX)
        m.append((1 << i) | (m[p] if p >= 0 else 0))
    return np.array(m, np.uint64).view(np.int64)


def tree_attn_scratch(n_heads, d, n_tok, batch, max_ctx):
    """Bytes of scratch a tree_attn_dev call of these sizes, or smaller ones, needs."""
    n = lib().dsv4b_tree_attn_scratch(_int(n_heads, "n_heads"), _int(d, "d"), _int(n_tok, "n_tok"), _int(batch, "batch"),
                                      _int(max_ctx, "max_ctx"))
    if n == 0:
        raise ValueError("sizes that dsv4b_tree_attn does not take")
    return n


def tree_attn_dev(o, q, cache, pages, ctx, n_draft, mask, sink, max_ctx, scale, scratch, stream=None):
    """Attention of drafted tokens q [batch, tokens, heads, d] (bfloat16 or
    float16) over the cache, into o (same type). pages [batch, max_pages],
    ctx [batch] and n_draft [batch] (or None) are int32, mask [batch, tokens]
    int64 (tree_mask), sink [heads] float32 or None, scratch at least
    tree_attn_scratch() bytes that no other call uses meanwhile."""
    dev, shape = cache.device, q.shape
    if len(shape) != 4 or o.shape != shape or o.dtype is not q.dtype or shape[3] != cache.d:
        raise ValueError("q and o must be [batch, tokens, heads, d] of one type")
    b, t, h, d = shape
    tok = []
    for x, what in ((o, "o"), (q, "q")):
        s = x.stride()
        if x.get_device() != dev or s[3] != 1 or (h > 1 and s[2] != d):
            raise ValueError("%s must have contiguous heads on the cache's device" % what)
        st = s[1] if t > 1 else (s[0] if b > 1 else h * d)
        if b > 1 and s[0] != t * st:
            raise ValueError("%s: the tokens of all sequences must be evenly spaced" % what)
        tok.append(st)
    if pages.dim() != 2 or pages.shape[0] != b:
        raise ValueError("pages must be [batch, max_pages]")
    max_ctx = int(max_ctx)
    if (b | t | h | max_ctx | pages.shape[1]) >> 31:
        _too_long()
    if scratch.get_device() != dev or not scratch.is_contiguous():
        raise ValueError("scratch must be contiguous, on the cache's device")
    i32 = _t.int32
    _enqueue(lib().dsv4b_tree_attn, "dsv4b_tree_attn", dev, o.data_ptr(), q.data_ptr(), _dt(q, "q"), tok[0], tok[1],
             cache.ref, _want(pages, "pages", dev, i32), pages.shape[1], _want(ctx, "ctx", dev, i32, (b,)),
             None if n_draft is None else _want(n_draft, "n_draft", dev, i32, (b,)),
             _want(mask, "mask", dev, _t.int64, (b, t)),
             None if sink is None else _want(sink, "sink", dev, _t.float32, (h,)), h, t, b, max_ctx,
             float(scale), scratch.data_ptr(), scratch.numel() * scratch.element_size(),
             _stream(dev, stream, (o, q, cache.codes, cache.scales, pages, ctx, n_draft, mask, sink, scratch)))


def tree_attn_status(device=None):
    """Waits for the device (the current one for None); True when every
    tree_attn_dev there since the last status has run to its end. False: one of
    them gave up a wait inside the kernel, and its output is not valid."""
    _torch()
    with _t.cuda.device(device):
        rc = lib().dsv4b_tree_attn_status()
    if rc < 0:
        raise RuntimeError("dsv4b_tree_attn_status failed (rc=%d)" % rc)
    return rc == 0


class LogitAdjust:
    """What logits_dev does to each row (dsv4b_logit_adjust); the tensors are
    kept, and may be rewritten between calls. hist [rows, n] int32 token ids
    with hist_len and n_prompt [rows] int32; rep, freq, pres [rows] float32;
    bias_ids int32 and bias float32 [rows, n] with bias_len [rows] int32; mask
    [rows, words] int32, one bit per token."""

    def __init__(self, hist=None, hist_len=None, n_prompt=None, rep=None, freq=None, pres=None, bias_ids=None,
                 bias=None, bias_len=None, mask=None):
        if hist is not None and hist.shape[-1] == 0:      # no history at all
            hist = hist_len = n_prompt = rep = freq = pres = None
        if bias is not None and bias.shape[-1] == 0:
            bias = bias_ids = bias_len = None
        given = [t for t in (hist, bias, mask) if t is not None]
        self.rows = given[0].shape[0] if given else None
        self.device = given[0].get_device() if given else None
        if given and self.device < 0:
            raise ValueError("the tensors must be on a CUDA device")
        if (hist is None) != (hist_len is None) or (bias is None) != (bias_ids is None) or \
                (bias is None) != (bias_len is None):
            raise ValueError("hist goes with hist_len, bias with bias_ids and bias_len")
        if hist is None and any(t is not None for t in (n_prompt, rep, freq, pres)):
            raise ValueError("penalties need hist")
        two = [t for t in (hist, bias_ids, bias, mask) if t is not None]
        if any(t.dim() != 2 or t.shape[0] != self.rows for t in two):
            raise ValueError("hist, bias_ids, bias and mask must be [rows, n]")
        if bias is not None and bias.shape != bias_ids.shape:
            raise ValueError("bias and bias_ids must have one shape")
        i32, f32 = _torch().int32, _torch().float32

        def want(t, what, dtype, shape=None):
            return None if t is None else _want(t, what, self.device, dtype, shape)

        r = (self.rows,)
        self.keep = (hist, hist_len, n_prompt, rep, freq, pres, bias_ids, bias, bias_len, mask)
        self.c = LogitAdjustC(
            want(hist, "hist", i32), 0 if hist is None else hist.shape[1], want(hist_len, "hist_len", i32, r),
            want(n_prompt, "n_prompt", i32, r), want(rep, "rep", f32, r), want(freq, "freq", f32, r),
            want(pres, "pres", f32, r), want(bias_ids, "bias_ids", i32), want(bias, "bias", f32),
            0 if bias is None else bias.shape[1], want(bias_len, "bias_len", i32, r), want(mask, "mask", i32),
            0 if mask is None else mask.shape[1])
        self.ref = C.addressof(self.c)


def logits_dev(out, x, token, adjust=None, stream=None):
    """Adjusted logits of x [rows, vocab] into out (None: not wanted; may be
    x), and the greedy tokens into token [rows] (int32, or None)."""
    i32 = _torch().int32
    dev, shape, xs = x.get_device(), x.shape, x.stride()
    if len(shape) != 2 or xs[1] != 1 or dev < 0:
        raise ValueError("x must be a CUDA tensor [rows, vocab] with unit-stride rows")
    r, v = shape
    if (r | v) >> 31:
        _too_long()
    po = so = 0
    if out is not None:
        so = out.stride()
        if out.shape != shape or out.dtype is not x.dtype or out.get_device() != dev or so[1] != 1:
            raise ValueError("out must be like x")
        po, so = out.data_ptr(), so[0] if r > 1 else v
    if adjust is not None and adjust.rows is not None and (adjust.rows != r or adjust.device != dev):
        raise ValueError("the adjustments are for other rows or another device")
    _enqueue(lib().dsv4b_logits, "dsv4b_logits", dev, po, x.data_ptr(), _dt(x, "x"), so, xs[0] if r > 1 else v,
             None if token is None else _want(token, "token", dev, i32, (r,)), None if adjust is None else adjust.ref,
             r, v, _stream(dev, stream, (out, x, token) + (adjust.keep if adjust is not None else ())))


# ------------------------------------------------------------- whole model

def nccl_unique_id():
    """A new communicator id (bytes) for a sharded model; rank 0 makes it and
    every rank passes the same bytes to Model(..., nccl_id=...)."""
    buf = C.create_string_buffer(lib().dsv4b_nccl_id_bytes())
    check(lib().dsv4b_nccl_unique_id(buf), "dsv4b_nccl_unique_id")
    return buf.raw


def shard_check(cfg, world):
    """True when a model of ctypes config cfg splits over world GPUs."""
    return lib().dsv4b_shard_check(C.addressof(cfg), int(world)) == 0


# the split dimensions of dsv4b_shard_plan, in its order
SHARD_DIMS = ("heads", "q_rows", "o_groups", "o_lora", "inter", "shared_inter", "vocab")


def shard_plan(cfg, world, rank):
    """{dimension: (first, count)} of rank's share of each split dimension
    (dsv4b_shard_plan), or None when cfg does not split over world GPUs."""
    out = (C.c_int * (2 * len(SHARD_DIMS)))()
    if lib().dsv4b_shard_plan(C.addressof(cfg), int(world), int(rank), out) != len(SHARD_DIMS):
        return None
    return {k: (out[2 * j], out[2 * j + 1]) for j, k in enumerate(SHARD_DIMS)}


class Model:
    """A whole model resident on the device (dsv4_cuda_model_create) from a
    dsv4_model.SyntheticModel or any holder of cfg/mw/layers/experts structs.
    With world > 1 (synthetic only), this rank's share of a model sharded over
    world GPUs (one process per GPU, all stepping in lockstep). With n_seq > 1
    (one GPU), a batch of n_seq sequences stepped together
    (generate_batch / begin_batch / decode_batch)."""

    def __init__(self, sm, max_pos, synthetic_seed=None, rank=0, world=1, nccl_id=None, n_seq=1):
        """sm: a dsv4_model.SyntheticModel (host weights), or with
        synthetic_seed set, any holder of .cfg/.d for an on-device model."""
        self.sm, self.max_pos, self.n_seq = sm, max_pos, n_seq
        self.vocab = sm.d["vocab"]
        if n_seq != 1 and world != 1:
            raise ValueError("a batched model runs on one GPU")
        if synthetic_seed is None:
            if world != 1:
                raise ValueError("sharded models are synthetic (synthetic_seed)")
            self.h = lib().dsv4_cuda_model_create_batch(C.addressof(sm.cfg), C.addressof(sm.mw),
                                                        C.addressof(sm.layers), C.addressof(sm.experts), max_pos,
                                                        int(n_seq))
        elif world == 1:
            self.h = lib().dsv4_cuda_model_create_synthetic_batch(C.addressof(sm.cfg), max_pos, synthetic_seed,
                                                                  int(n_seq))
        else:
            idb = C.create_string_buffer(bytes(nccl_id), len(nccl_id))
            self.h = lib().dsv4_cuda_model_create_synthetic_sharded(C.addressof(sm.cfg), max_pos, synthetic_seed,
                                                                    int(rank), int(world), idb)
        if not self.h:
            raise RuntimeError("model creation failed")

    def decode(self, token, pos):
        nxt = np.zeros(1, np.int32)
        check(lib().dsv4_cuda_model_decode(self.h, int(token), int(pos), nxt.ctypes.data),
              "dsv4_cuda_model_decode")
        return int(nxt[0])

    def device_bytes(self):
        return lib().dsv4_cuda_model_bytes(self.h)

    def begin(self, prompt):
        p = np.ascontiguousarray(prompt, np.int32)
        check(lib().dsv4_cuda_model_begin(self.h, p.ctypes.data, p.size), "dsv4_cuda_model_begin")

    def step(self, want_logits=False):
        tok = np.zeros(1, np.int32)
        lg = np.empty(self.vocab, np.float32) if want_logits else None
        check(lib().dsv4_cuda_model_step(self.h, tok.ctypes.data, None if lg is None else lg.ctypes.data),
              "dsv4_cuda_model_step")
        return int(tok[0]), lg

    def generate(self, prompt, n_gen):
        p = np.ascontiguousarray(prompt, np.int32)
        out = np.empty(n_gen + 1, np.int32)
        n = lib().dsv4_cuda_model_generate(self.h, p.ctypes.data, p.size, n_gen, out.ctypes.data)
        if n < 0:
            raise RuntimeError("dsv4_cuda_model_generate failed")
        return out[:n]

    def prefill(self, prompt, chunk=32):
        """The prompt in passes of chunk tokens; returns the first generated
        token. Steps continue from position len(prompt)."""
        p = np.ascontiguousarray(prompt, np.int32)
        tok = lib().dsv4b_model_prefill(self.h, p.ctypes.data, p.size, int(chunk))
        if tok < 0:
            raise RuntimeError("dsv4b_model_prefill failed")
        return tok

    def generate_prefill(self, prompt, n_gen, chunk=32):
        """generate() with the prompt prefilled in passes of chunk tokens."""
        p = np.ascontiguousarray(prompt, np.int32)
        out = np.empty(n_gen + 1, np.int32)
        n = lib().dsv4b_model_generate_prefill(self.h, p.ctypes.data, p.size, n_gen, int(chunk), out.ctypes.data)
        if n < 0:
            raise RuntimeError("dsv4b_model_generate_prefill failed")
        return out[:n]

    def begin_batch(self, prompts):
        """prompts: [n_seq][n_prompt] int32, one row per sequence."""
        p = np.ascontiguousarray(prompts, np.int32)
        if p.ndim != 2 or p.shape[0] != self.n_seq:
            raise ValueError("prompts must be [n_seq][n_prompt]")
        check(lib().dsv4b_model_begin_batch(self.h, p.ctypes.data, p.shape[1]), "dsv4b_model_begin_batch")

    def generate_batch(self, prompts, n_gen):
        """Greedy tokens [n_seq][n_gen + 1] of every sequence, from its last
        prompt position on."""
        p = np.ascontiguousarray(prompts, np.int32)
        if p.ndim != 2 or p.shape[0] != self.n_seq:
            raise ValueError("prompts must be [n_seq][n_prompt]")
        out = np.empty((self.n_seq, n_gen + 1), np.int32)
        n = lib().dsv4b_model_generate_batch(self.h, p.ctypes.data, p.shape[1], n_gen, out.ctypes.data)
        if n < 0:
            raise RuntimeError("dsv4b_model_generate_batch failed")
        return out[:, :n]

    def decode_batch(self, tokens, pos):
        """Every sequence's token at pos in (host), the next tokens out."""
        t = np.ascontiguousarray(tokens, np.int32)
        nxt = np.zeros(self.n_seq, np.int32)
        check(lib().dsv4b_model_decode_batch(self.h, t.ctypes.data, int(pos), nxt.ctypes.data),
              "dsv4b_model_decode_batch")
        return nxt

    def step_async(self, stream=None):
        check(lib().dsv4b_model_step_async(self.h, stream_ptr(stream)), "dsv4b_model_step_async")

    def close(self):
        if self.h:
            lib().dsv4_cuda_model_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
