"""ctypes binding of libapoe.so (the C-ABI declared in include/apoe.h).

Arrays may be numpy arrays (host) or torch tensors (host or the context's GPU); the
library copies as needed. There is no CPU fallback: if the HIP library is missing or a
call fails, an exception is raised.

The operators that fit a query adapter (`softmax_loss`, `orthogonalize`, `gated_residual`) and those that its layers are built and trained
from (`embed`, `layer_norm`, `linear`, `AdamW`) take torch tensors on the context's GPU, write torch tensors and return without waiting; their
work is ordered with torch's current stream.
"""
import ctypes as C
import os
import sys

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libapoe.so")

INF_DIS = 1000000.0
KW_SLOTS = 8
KW_CAND = 32
WITHOUT_CODES, WITHOUT_SKETCHES = 1, 2

_lib = None


class ApoeError(RuntimeError):
    pass


class SearchParams(C.Structure):
    _fields_ = [("w_dense", C.c_float), ("w_sparse", C.c_float), ("w_bm25", C.c_float), ("kg_weight", C.c_float),
                ("cands", C.c_uint32), ("max_iter", C.c_uint32), ("q_begin", C.c_uint32), ("q_count", C.c_uint32),
                ("variant", C.c_uint32), ("keyword_filter", C.c_uint32)]


class SearchStats(C.Structure):
    _fields_ = [("kernel_ms", C.c_float), ("expansions", C.c_uint64), ("evaluations", C.c_uint64),
                ("nnz_sparse", C.c_uint64), ("nnz_bm25", C.c_uint64), ("dense_rows", C.c_uint64), ("algo_bytes", C.c_uint64)]


class SoftmaxLossArgs(C.Structure):
    _fields_ = [("dtype", C.c_uint32), ("n_queries", C.c_uint32), ("n_rows", C.c_uint32), ("dim", C.c_uint32),
                ("q", C.c_void_p), ("rows", C.c_void_p), ("corpus", C.c_void_p),
                ("q_stride", C.c_uint64), ("rows_stride", C.c_uint64), ("grad_q_stride", C.c_uint64), ("grad_rows_stride", C.c_uint64),
                ("t_off", C.c_void_p), ("t_idx", C.c_void_p), ("t_val", C.c_void_p), ("live", C.c_void_p), ("weight", C.c_void_p),
                ("scale", C.c_float), ("loss", C.c_void_p), ("lse", C.c_void_p), ("grad_q", C.c_void_p), ("grad_rows", C.c_void_p)]


class OrthogonalizeArgs(C.Structure):
    _fields_ = [("in_dtype", C.c_uint32), ("out_dtype", C.c_uint32), ("products", C.c_uint32),
                ("batch", C.c_uint32), ("rows", C.c_uint32), ("cols", C.c_uint32),
                ("in_stride", C.c_uint64), ("out_stride", C.c_uint64), ("in_batch_stride", C.c_uint64), ("out_batch_stride", C.c_uint64),
                ("in_", C.c_void_p), ("out", C.c_void_p), ("steps", C.c_uint32),
                ("a", C.c_float), ("b", C.c_float), ("c", C.c_float), ("alpha", C.c_float), ("beta", C.c_float)]


class GatedResidualArgs(C.Structure):
    _fields_ = [("dtype", C.c_uint32), ("rows", C.c_uint32), ("dim", C.c_uint32), ("gate_kind", C.c_uint32),
                ("x_stride", C.c_uint64), ("h_stride", C.c_uint64), ("gate_stride", C.c_uint64), ("y_stride", C.c_uint64), ("u_stride", C.c_uint64),
                ("x", C.c_void_p), ("h", C.c_void_p), ("gate", C.c_void_p), ("scale", C.c_void_p), ("w_post", C.c_void_p), ("w_next", C.c_void_p),
                ("eps", C.c_float), ("y", C.c_void_p), ("u", C.c_void_p),
                ("grad_y_stride", C.c_uint64), ("grad_u_stride", C.c_uint64), ("grad_x_stride", C.c_uint64), ("grad_h_stride", C.c_uint64), ("grad_gate_stride", C.c_uint64),
                ("grad_y", C.c_void_p), ("grad_u", C.c_void_p), ("grad_x", C.c_void_p), ("grad_h", C.c_void_p), ("grad_gate", C.c_void_p),
                ("grad_scale", C.c_void_p), ("grad_w_post", C.c_void_p), ("grad_w_next", C.c_void_p)]


class EmbedArgs(C.Structure):
    _fields_ = [("dtype", C.c_uint32), ("n_rows", C.c_uint32), ("n_table", C.c_uint32), ("n_entries", C.c_uint32), ("dim", C.c_uint32),
                ("table", C.c_void_p), ("idx", C.c_void_p), ("off", C.c_void_p), ("val", C.c_void_p), ("scale", C.c_float), ("base", C.c_void_p), ("out", C.c_void_p),
                ("table_stride", C.c_uint64), ("base_stride", C.c_uint64), ("out_stride", C.c_uint64),
                ("grad", C.c_void_p), ("grad_table", C.c_void_p), ("grad_val", C.c_void_p), ("grad_stride", C.c_uint64), ("grad_table_stride", C.c_uint64),
                ("accumulate", C.c_uint32)]


class LayerNormArgs(C.Structure):
    _fields_ = [("dtype", C.c_uint32), ("rows", C.c_uint32), ("dim", C.c_uint32), ("x", C.c_void_p), ("w", C.c_void_p), ("b", C.c_void_p), ("eps", C.c_float),
                ("y", C.c_void_p), ("x_stride", C.c_uint64), ("y_stride", C.c_uint64),
                ("grad_y_stride", C.c_uint64), ("grad_skip_stride", C.c_uint64), ("grad_x_stride", C.c_uint64),
                ("grad_y", C.c_void_p), ("grad_skip", C.c_void_p), ("grad_x", C.c_void_p), ("grad_w", C.c_void_p), ("grad_b", C.c_void_p)]


class LinearArgs(C.Structure):
    _fields_ = [("dtype", C.c_uint32), ("rows", C.c_uint32), ("cols_in", C.c_uint32), ("cols_out", C.c_uint32), ("act", C.c_uint32),
                ("x", C.c_void_p), ("w", C.c_void_p), ("bias", C.c_void_p), ("residual", C.c_void_p), ("y", C.c_void_p), ("pre", C.c_void_p),
                ("x_stride", C.c_uint64), ("w_stride", C.c_uint64), ("residual_stride", C.c_uint64), ("y_stride", C.c_uint64), ("pre_stride", C.c_uint64),
                ("grad_y", C.c_void_p), ("grad_x", C.c_void_p), ("grad_w", C.c_void_p), ("grad_bias", C.c_void_p),
                ("grad_y_stride", C.c_uint64), ("grad_x_stride", C.c_uint64), ("grad_w_stride", C.c_uint64)]


class AdamwTensor(C.Structure):
    _fields_ = [("p", C.c_void_p), ("m", C.c_void_p), ("v", C.c_void_p), ("m_scale", C.c_void_p), ("v_scale", C.c_void_p), ("copy", C.c_void_p),
                ("copy_dtype", C.c_uint32), ("n", C.c_uint64), ("decay", C.c_double)]


class AdamwStepArgs(C.Structure):
    _fields_ = [("grads", C.c_void_p), ("grad_dtypes", C.c_void_p), ("lr", C.c_double), ("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double),
                ("grad_scale", C.c_double), ("step", C.c_uint32), ("step_dev", C.c_void_p), ("lr_dev", C.c_void_p), ("step_taken", C.c_void_p)]


EXPORTS = [
    "apoe_last_error_string", "apoe_ctx_create", "apoe_ctx_destroy", "apoe_ctx_synchronize", "apoe_corpus_create", "apoe_corpus_create_without",
    "apoe_corpus_destroy", "apoe_corpus_info", "apoe_corpus_bytes", "apoe_corpus_pair_bytes", "apoe_corpus_make_half_rows", "apoe_queries_create", "apoe_queries_destroy",
    "apoe_kg_create", "apoe_kg_destroy", "apoe_calibrate_weights", "apoe_hybrid_distance_batch", "apoe_hybrid_distance_pairs", "apoe_norms",
    "apoe_knn_create", "apoe_knn_destroy", "apoe_knn_use_half_rows", "apoe_knn_set_join", "apoe_nnd_init", "apoe_nnd_iterate", "apoe_nnd_merge_reverse",
    "apoe_knn_download", "apoe_knn_upload", "apoe_knn_download_reverse", "apoe_knn_upload_reverse", "apoe_knn_set_prune_form", "apoe_prune", "apoe_prune_download", "apoe_finalize_graph",
    "apoe_knn_elapsed_ms", "apoe_knn_counters", "apoe_knn_read_counters", "apoe_graph_create", "apoe_graph_destroy", "apoe_graph_info", "apoe_graph_download",
    "apoe_search", "apoe_search_noalloc",
    "apoe_ctx_create_on_stream", "apoe_ctx_stream", "apoe_softmax_loss", "apoe_orthogonalize", "apoe_gated_residual", "apoe_gated_residual_grad",
    "apoe_embed", "apoe_embed_grad", "apoe_layer_norm", "apoe_layer_norm_grad", "apoe_linear", "apoe_linear_grad",
    "apoe_adamw_create", "apoe_adamw_destroy", "apoe_adamw_step", "apoe_adamw_moments",
]


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ApoeError(f"{LIB_PATH} is not built; run `make -C {os.path.join(_HERE, 'csrc')}`")
        # PyTorch wheels bring their own copy of the HIP runtime. A process that loads this library
        # first and PyTorch second ends up with two runtimes, and the second one finds no device:
        # let PyTorch (if it is installed) load its copy first, libapoe.so then binds to the same one.
        if "torch" not in sys.modules:
            try:
                import torch  # noqa: F401
            except ImportError:
                pass
        _lib = C.CDLL(LIB_PATH)
        _lib.apoe_last_error_string.restype = C.c_char_p
        _lib.apoe_corpus_bytes.restype = C.c_uint64
        _lib.apoe_corpus_bytes.argtypes = [C.c_void_p]
        _lib.apoe_corpus_pair_bytes.restype = C.c_uint32
        _lib.apoe_corpus_pair_bytes.argtypes = [C.c_void_p]
        _lib.apoe_knn_elapsed_ms.restype = C.c_float
        _lib.apoe_knn_elapsed_ms.argtypes = [C.c_void_p]
        for name in ("apoe_ctx_destroy", "apoe_corpus_destroy", "apoe_queries_destroy", "apoe_kg_destroy",
                     "apoe_knn_destroy", "apoe_graph_destroy", "apoe_adamw_destroy"):
            getattr(_lib, name).restype = None
            getattr(_lib, name).argtypes = [C.c_void_p]
    return _lib


def _check(status):
    if status != 0:
        raise ApoeError(f"apoe status {status}: {lib().apoe_last_error_string().decode()}")


def _ptr(a, dtype):
    """(keepalive, void*) of a numpy array or torch tensor of the given numpy dtype."""
    if a is None:
        return None, C.c_void_p(0)
    if isinstance(a, np.ndarray):
        if a.dtype != dtype or not a.flags.c_contiguous:
            a = np.ascontiguousarray(a, dtype=dtype)
        return a, C.c_void_p(a.ctypes.data)
    import torch
    want = {np.dtype(np.float32): torch.float32, np.dtype(np.uint32): (torch.int32, torch.uint32)}[np.dtype(dtype)]
    if isinstance(want, tuple):
        assert a.dtype in want, a.dtype
    else:
        assert a.dtype == want, a.dtype
    a = a.contiguous()
    return a, C.c_void_p(a.data_ptr())


class Context:
    """stream: a torch stream (or the integer of a HIP stream) that the context's work is put on; by default it has a stream
    of its own."""

    def __init__(self, device=0, stream=None):
        self.h = C.c_void_p()
        if stream is None:
            _check(lib().apoe_ctx_create(C.c_int(device), C.byref(self.h)))
        else:
            self._stream_kept = stream  # outlives the context
            handle = int(getattr(stream, "cuda_stream", stream))
            _check(lib().apoe_ctx_create_on_stream(C.c_int(device), C.c_void_p(handle), C.byref(self.h)))
        out = C.c_void_p()
        _check(lib().apoe_ctx_stream(self.h, C.byref(out)))
        self.stream = out.value or 0
        self._torch_stream = None
        self.device = device

    def synchronize(self):
        _check(lib().apoe_ctx_synchronize(self.h))

    def torch_stream(self):
        """The context's stream as torch sees it."""
        if self._torch_stream is None:
            import torch
            self._torch_stream = torch.cuda.ExternalStream(self.stream, device=self.device) if self.stream else torch.cuda.default_stream(self.device)
        return self._torch_stream

    def close(self):
        if self.h:
            lib().apoe_ctx_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Corpus:
    def __init__(self, ctx, dense, s_off, s_idx, s_val, b_off, b_idx, b_val, without=0):
        self.ctx = ctx
        n, dim = dense.shape
        keep = [_ptr(dense, np.float32), _ptr(s_off, np.uint32), _ptr(s_idx, np.uint32), _ptr(s_val, np.float32),
                _ptr(b_off, np.uint32), _ptr(b_idx, np.uint32), _ptr(b_val, np.float32)]
        self.h = C.c_void_p()
        _check(lib().apoe_corpus_create_without(ctx.h, C.c_uint32(without), C.c_uint32(n), C.c_uint32(dim), *[k[1] for k in keep], C.byref(self.h)))
        self.n, self.dim = n, dim

    def info(self):
        out = (C.c_uint32 * 4)()
        _check(lib().apoe_corpus_info(self.h, out))
        return list(out)

    def bytes(self):
        return int(lib().apoe_corpus_bytes(self.h))

    def pair_bytes(self):
        return int(lib().apoe_corpus_pair_bytes(self.h))

    def make_half_rows(self):
        """Half-precision copy of the dense rows, for searches with variant | 0x200."""
        _check(lib().apoe_corpus_make_half_rows(self.ctx.h, self.h))

    def close(self):
        if self.h:
            lib().apoe_corpus_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Queries:
    def __init__(self, ctx, dense, s_off, s_idx, s_val, b_off, b_idx, b_val):
        self.ctx = ctx
        n, dim = dense.shape
        keep = [_ptr(dense, np.float32), _ptr(s_off, np.uint32), _ptr(s_idx, np.uint32), _ptr(s_val, np.float32),
                _ptr(b_off, np.uint32), _ptr(b_idx, np.uint32), _ptr(b_val, np.float32)]
        self.h = C.c_void_p()
        _check(lib().apoe_queries_create(ctx.h, C.c_uint32(n), C.c_uint32(dim), *[k[1] for k in keep], C.byref(self.h)))
        self.n, self.dim = n, dim

    def close(self):
        if self.h:
            lib().apoe_queries_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class KnowledgeGraph:
    def __init__(self, ctx, e2e_off, e2e_idx, e2d_off, e2d_idx, q2e_off, q2e_idx):
        self.ctx = ctx
        keep = [_ptr(a, np.uint32) for a in (e2e_off, e2e_idx, e2d_off, e2d_idx)]
        keepq = [_ptr(a, np.uint32) for a in (q2e_off, q2e_idx)]
        self.h = C.c_void_p()
        _check(lib().apoe_kg_create(ctx.h, C.c_uint32(len(e2e_off) - 1), *[k[1] for k in keep], C.c_uint32(len(q2e_off) - 1),
                                    *[k[1] for k in keepq], C.byref(self.h)))

    def close(self):
        if self.h:
            lib().apoe_kg_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Graph:
    def __init__(self, ctx, rows=None, entry=None, handle=None):
        self.ctx = ctx
        if handle is not None:
            self.h = handle
        else:
            n, W = rows.shape
            kr, ke = _ptr(rows, np.uint32), _ptr(entry, np.uint32)
            self.h = C.c_void_p()
            _check(lib().apoe_graph_create(ctx.h, C.c_uint32(n), C.c_uint32(W), kr[1], ke[1], C.c_uint32(len(entry)), C.byref(self.h)))
        info = (C.c_uint32 * 3)()
        _check(lib().apoe_graph_info(self.h, info))
        self.n, self.width, self.n_entry = info[0], info[1], info[2]

    def download(self):
        rows = np.empty((self.n, self.width), np.uint32)
        entry = np.empty(self.n_entry, np.uint32)
        _check(lib().apoe_graph_download(self.h, C.c_void_p(rows.ctypes.data), C.c_void_p(entry.ctypes.data)))
        return rows, entry

    def close(self):
        if self.h:
            lib().apoe_graph_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Knn:
    """NN-Descent state and the build steps of index.cu:889-903."""

    def __init__(self, ctx, corpus, K=64, dense_scale=7.0):
        self.ctx, self.corpus, self.K = ctx, corpus, K
        self.h = C.c_void_p()
        _check(lib().apoe_knn_create(ctx.h, corpus.h, C.c_uint32(K), C.c_float(dense_scale), C.byref(self.h)))
        self.degree = None

    def use_half_rows(self, on=True):
        """NN-Descent steps on the half-precision rows; merge_reverse() then recomputes the stored distances in fp32."""
        _check(lib().apoe_knn_use_half_rows(self.h, C.c_int(1 if on else 0)))

    def set_join(self, mode):
        """0: the reference's expansion step; 1: local join around the picked neighbour; 2: the same, both endpoints updated."""
        _check(lib().apoe_knn_set_join(self.h, C.c_int(mode)))

    def init(self, seed):
        _check(lib().apoe_nnd_init(self.h, C.c_uint64(seed)))

    def iterate(self, last=False):
        ins = C.c_uint64(0)
        _check(lib().apoe_nnd_iterate(self.h, C.c_int(1 if last else 0), C.byref(ins)))
        return ins.value

    def merge_reverse(self):
        _check(lib().apoe_nnd_merge_reverse(self.h))

    def download(self):
        ids = np.empty((self.corpus.n, self.K), np.uint32)
        dist = np.empty((self.corpus.n, self.K), np.float32)
        _check(lib().apoe_knn_download(self.h, C.c_void_p(ids.ctypes.data), C.c_void_p(dist.ctypes.data)))
        return ids, dist

    def upload(self, ids, dist):
        ki, kd = _ptr(ids, np.uint32), _ptr(dist, np.float32)
        _check(lib().apoe_knn_upload(self.h, ki[1], kd[1]))

    def download_reverse(self):
        """(rev_ids [n][K], rev_dist [n][K], rev_cnt [n]): the reverse lists as they stand."""
        ids = np.empty((self.corpus.n, self.K), np.uint32)
        dist = np.empty((self.corpus.n, self.K), np.float32)
        cnt = np.empty(self.corpus.n, np.uint32)
        _check(lib().apoe_knn_download_reverse(self.h, C.c_void_p(ids.ctypes.data), C.c_void_p(dist.ctypes.data), C.c_void_p(cnt.ctypes.data)))
        return ids, dist, cnt

    def upload_reverse(self, rev_ids, rev_dist, rev_cnt):
        ri, rd, rc = _ptr(rev_ids, np.uint32), _ptr(rev_dist, np.float32), _ptr(rev_cnt, np.uint32)
        _check(lib().apoe_knn_upload_reverse(self.h, ri[1], rd[1], rc[1]))

    def set_prune_form(self, form):
        """0: the gather-once forms of the prune where they apply (default); 1: the table-probing kernel."""
        _check(lib().apoe_knn_set_prune_form(self.h, C.c_int(form)))

    def prune(self, degree):
        _check(lib().apoe_prune(self.h, C.c_uint32(degree)))
        self.degree = degree

    def prune_download(self):
        n, d = self.corpus.n, self.degree
        fwd = np.empty((n, d), np.uint32)
        det = np.empty((n, d), np.uint32)
        cnt = np.empty(n, np.uint32)
        kw = np.empty((n, 1 + KW_CAND), np.uint32)
        _check(lib().apoe_prune_download(self.h, *[C.c_void_p(a.ctypes.data) for a in (fwd, det, cnt, kw)]))
        return fwd, det, cnt, kw

    def finalize(self):
        h = C.c_void_p()
        _check(lib().apoe_finalize_graph(self.h, C.byref(h)))
        return Graph(self.ctx, handle=h)

    def elapsed_ms(self):
        return float(lib().apoe_knn_elapsed_ms(self.h))

    def counters(self):
        """(evaluations, dense rows read) of the NN-Descent steps since init."""
        out = (C.c_uint64 * 2)()
        _check(lib().apoe_knn_counters(self.h, out))
        return int(out[0]), int(out[1])

    def read_counters(self):
        """(dense rows, rows of pairs, sketches) that the NN-Descent steps since init read."""
        out = (C.c_uint64 * 3)()
        _check(lib().apoe_knn_read_counters(self.h, out))
        return int(out[0]), int(out[1]), int(out[2])

    def close(self):
        if self.h:
            lib().apoe_knn_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def build_graph(ctx, corpus, K=64, iters=25, degree=32, dense_scale=7.0, seed=1, half_rows=False, join=0, expansion_first=0):
    """NN-Descent + reverse merge + prune + final assembly; returns (Graph, gpu_ms). With a join mode, the first
    `expansion_first` steps are expansion steps all the same (on very large corpora one such step gets the lists going)."""
    knn = Knn(ctx, corpus, K, dense_scale)
    if half_rows:
        corpus.make_half_rows()
        knn.use_half_rows()
    knn.init(seed)
    for it in range(iters):
        if join:
            knn.set_join(0 if it < expansion_first else join)
        knn.iterate(last=(it == iters - 1))
    knn.merge_reverse()
    knn.prune(degree)
    g = knn.finalize()
    ms = knn.elapsed_ms()
    knn.close()
    return g, ms


def distance_batch(ctx, corpus, queries, w3, ids):
    ids = np.ascontiguousarray(ids, np.uint32)
    assert ids.shape[0] == queries.n
    out = np.empty(ids.shape, np.float32)
    w = (C.c_float * 3)(*w3)
    _check(lib().apoe_hybrid_distance_batch(ctx.h, corpus.h, queries.h, w, C.c_void_p(ids.ctypes.data), C.c_uint32(ids.shape[1]),
                                            C.c_void_p(out.ctypes.data)))
    return out


def distance_pairs(ctx, corpus, dense_scale, a, b):
    a = np.ascontiguousarray(a, np.uint32)
    b = np.ascontiguousarray(b, np.uint32)
    out = np.empty(len(a), np.float32)
    _check(lib().apoe_hybrid_distance_pairs(ctx.h, corpus.h, C.c_float(dense_scale), C.c_void_p(a.ctypes.data),
                                            C.c_void_p(b.ctypes.data), C.c_uint32(len(a)), C.c_void_p(out.ctypes.data)))
    return out


def norms(ctx, corpus, dense_scale):
    out = np.empty(corpus.n, np.float32)
    _check(lib().apoe_norms(ctx.h, corpus.h, C.c_float(dense_scale), C.c_void_p(out.ctypes.data)))
    return out


def calibrate_weights(ctx, corpus, queries, w3, n_queries=None):
    """Effective (dense, sparse, bm25) weights after the reference's calibration step."""
    w = (C.c_float * 3)(*w3)
    _check(lib().apoe_calibrate_weights(ctx.h, corpus.h, queries.h, C.c_uint32(queries.n if n_queries is None else n_queries), w))
    return (float(w[0]), float(w[1]), float(w[2]))


def search(ctx, corpus, queries, graph, w3, cands, kg=None, kg_weight=0.0, max_iter=0, q_begin=0, q_count=0, variant=0,
           out_ids=None, out_dist=None, keyword_filter=False):
    """Returns (ids [q, cands] u32, dist [q, cands] f32, SearchStats). w3 = (dense, sparse, bm25).
    keyword_filter: rows hold only documents with a BM25 term that the query flags (bit 31 of the
    query's BM25 term id) as a required keyword."""
    nq = q_count if q_count else queries.n - q_begin
    if q_begin > queries.n or nq > queries.n - q_begin:
        raise ApoeError(f"query range of {nq} from {q_begin} beyond {queries.n} queries")
    if out_ids is None:
        out_ids = np.empty((nq, cands), np.uint32)
        out_dist = np.empty((nq, cands), np.float32)
    for arr, dt, name in ((out_ids, np.uint32, "out_ids"), (out_dist, np.float32, "out_dist")):
        # the library writes into these: a copy made here would be filled and thrown away
        if isinstance(arr, np.ndarray):
            if arr.dtype != dt or not arr.flags.c_contiguous or arr.shape != (nq, cands):
                raise ApoeError(f"{name} must be a C-contiguous {np.dtype(dt).name} array of shape {(nq, cands)}")
        elif not arr.is_contiguous() or tuple(arr.shape) != (nq, cands):
            raise ApoeError(f"{name} must be a contiguous tensor of shape {(nq, cands)}")
    ki, kd = _ptr(out_ids, np.uint32), _ptr(out_dist, np.float32)
    p = SearchParams(w3[0], w3[1], w3[2], kg_weight, cands, max_iter, q_begin, q_count, variant, 1 if keyword_filter else 0)
    st = SearchStats()
    _check(lib().apoe_search(ctx.h, corpus.h, queries.h, graph.h, kg.h if kg is not None else C.c_void_p(0), C.byref(p), ki[1], kd[1],
                             C.byref(st)))
    return out_ids, out_dist, st


def search_noalloc(ctx, corpus, queries, graph, w3, cands, out_ids, out_dist, kg=None, kg_weight=0.0, max_iter=0, q_begin=0, q_count=0,
                   variant=0, keyword_filter=False, want_stats=True):
    """apoe_search_noalloc: the search with a static device workspace; out_ids / out_dist are device tensors
    [q, cands] that the kernels write in place. Without stats the call does not wait for the GPU."""
    nq = q_count if q_count else queries.n - q_begin
    assert tuple(out_ids.shape) == (nq, cands) and tuple(out_dist.shape) == (nq, cands) and out_ids.is_contiguous() and out_dist.is_contiguous()
    ki, kd = _ptr(out_ids, np.uint32), _ptr(out_dist, np.float32)
    p = SearchParams(w3[0], w3[1], w3[2], kg_weight, cands, max_iter, q_begin, q_count, variant, 1 if keyword_filter else 0)
    st = SearchStats() if want_stats else None
    _check(lib().apoe_search_noalloc(ctx.h, corpus.h, queries.h, graph.h, kg.h if kg is not None else C.c_void_p(0), C.byref(p), ki[1], kd[1],
                                     C.byref(st) if want_stats else C.c_void_p(0)))
    return st


# ---- fitting a query adapter ----

COEFS = (3.4445, -4.7750, 2.0315)  # quintic of five steps that bring singular values from 1e-3 on to between 0.7 and 1.2
_torch = _DTYPES = _INTS = _FLOATS = _raw_stream = None


def _load_torch():
    global _torch, _DTYPES, _INTS, _FLOATS, _raw_stream
    import torch
    _torch = torch
    # the current stream's address: without an object around it where torch offers that (2 us less a call)
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)
    _DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    _INTS, _FLOATS = (torch.int32, torch.uint32), (torch.float32,)


def _dtype(t, name):
    if _torch is None:
        _load_torch()
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ApoeError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    return code


def _on_gpu(ctx, t, name):
    if t.get_device() != ctx.device:
        raise ApoeError(f"{name} must be on GPU {ctx.device}, the context's")


def _matrix(ctx, t, name, shape=None, dtype=None):
    """Checks a matrix whose rows are contiguous; returns its row stride."""
    have = t.shape
    if t.get_device() != ctx.device:
        raise ApoeError(f"{name} must be on GPU {ctx.device}, the context's")
    if len(have) != 2 or (shape is not None and have != shape):
        raise ApoeError(f"{name} must be a matrix{'' if shape is None else f' of shape {tuple(shape)}'}, not {tuple(have)}")
    if dtype is not None and t.dtype is not dtype:
        raise ApoeError(f"{name} must be {dtype}, not {t.dtype}")
    n, d = have
    row, col = t.stride()
    if col != 1 and d > 1:
        raise ApoeError(f"the rows of {name} must be contiguous")
    if n <= 1:
        return d
    if row < d:
        raise ApoeError(f"the rows of {name} overlap")
    return row


def _vector(ctx, t, name, n, dtypes):
    shape = t.shape
    if t.get_device() != ctx.device:
        raise ApoeError(f"{name} must be on GPU {ctx.device}, the context's")
    if t.dtype not in dtypes or len(shape) != 1 or (n is not None and shape[0] != n) or not t.is_contiguous():
        raise ApoeError(f"{name} must be a contiguous vector of {' or '.join(str(d) for d in dtypes)}{'' if n is None else f' of length {n}'}")
    return t.data_ptr()


def _call(ctx, function, args):
    """Calls `function`; the context's stream waits for torch's current stream, and that for the context's afterwards (nothing where
    they are one)."""
    if _raw_stream(ctx.device) == ctx.stream:
        _check(function(ctx.h, C.byref(args)))
        return
    _ordered(ctx, lambda: function(ctx.h, C.byref(args)))


def _ordered(ctx, call):
    if _raw_stream(ctx.device) == ctx.stream:
        _check(call())
        return
    theirs, ours = _torch.cuda.current_stream(ctx.device), ctx.torch_stream()
    ours.wait_stream(theirs)
    status = call()
    theirs.wait_stream(ours)
    _check(status)


def softmax_loss(ctx, queries, rows, t_off, t_idx, t_val=None, scale=1.0, weight=None, live=None, grad_queries=False, grad_rows=False):
    """Softmax cross entropy of queries [m, d] over the rows [n, d] (a matrix, or a Corpus with half-precision rows), and the
    gradients of sum(weight * loss). t_off, t_idx, t_val: CSR of each query's relevant rows and their weights (equal shares
    without); live: int32 bit mask of the rows that take part; scale: of the inner products. grad_queries, grad_rows: True, or a
    matrix to write to. Returns dict(loss [m], lse [m]) and the gradients asked for; the logits are never held."""
    a = SoftmaxLossArgs()
    a.dtype = _dtype(queries, "queries")
    a.q_stride = _matrix(ctx, queries, "queries")
    m, d = queries.shape
    a.n_queries, a.dim = m, d
    if isinstance(rows, Corpus):
        a.n_rows, a.corpus = rows.n, rows.h
        if d != rows.dim:
            raise ApoeError(f"queries of {d} columns against a corpus of {rows.dim}")
        if grad_rows is not False and grad_rows is not None:
            raise ApoeError("the rows of a corpus stay as they are: no grad_rows")
    else:
        a.rows_stride = _matrix(ctx, rows, "rows", (len(rows), d), queries.dtype)
        a.n_rows, a.rows = rows.shape[0], rows.data_ptr()
        if rows.shape[0] == 0:
            raise ApoeError("rows is empty")
    a.t_off = _vector(ctx, t_off, "t_off", m + 1, _INTS)
    a.t_idx = _vector(ctx, t_idx, "t_idx", None, _INTS)
    if t_idx.numel() == 0:  # no target at all: no entry is read, but the pointer has to be one
        a.t_idx = a.t_off
    if t_val is not None:
        a.t_val = _vector(ctx, t_val, "t_val", t_idx.shape[0], _FLOATS) if t_idx.numel() else None
    if live is not None:
        a.live = _vector(ctx, live, "live", (a.n_rows + 31) // 32, _INTS)
    if weight is not None:
        a.weight = _vector(ctx, weight, "weight", m, _FLOATS)
    a.scale = scale
    a.q = queries.data_ptr()
    both = _torch.empty((2, m), dtype=_torch.float32, device=queries.device)
    out = dict(loss=both[0], lse=both[1])
    a.loss = both.data_ptr()
    a.lse = a.loss + 4 * m if m else a.loss
    if grad_queries is not False and grad_queries is not None:
        g = _torch.empty((m, d), dtype=queries.dtype, device=queries.device) if grad_queries is True else grad_queries
        a.grad_q_stride = _matrix(ctx, g, "grad_queries", (m, d), queries.dtype)
        out["grad_queries"], a.grad_q = g, g.data_ptr()
    if grad_rows is not False and grad_rows is not None:
        g = _torch.empty((rows.shape[0], d), dtype=rows.dtype, device=rows.device) if grad_rows is True else grad_rows
        a.grad_rows_stride = _matrix(ctx, g, "grad_rows", rows.shape, rows.dtype)
        out["grad_rows"], a.grad_rows = g, g.data_ptr()
    if m == 0:  # nothing to compute but a gradient of zeros
        if "grad_rows" in out:
            out["grad_rows"].zero_()
        return out
    _call(ctx, lib().apoe_softmax_loss, a)
    return out


def orthogonalize(ctx, x, out=None, steps=5, coefs=COEFS, alpha=1.0, beta=0.0, products=None):
    """out = alpha NS(x) + beta out for a matrix or a batch of matrices: the Newton-Schulz steps that bring x's singular values to
    about one. products: "f16" (1e-4 to 6e-4 of the result; a short side of up to 64 is exact to 1e-6 either way) or "f32"; by default "f16" where out is bfloat16.
    Coefficients under which an entry of X, A or (off its diagonal) b A + c A A passes 15 give a result that is not finite."""
    if x.dim() not in (2, 3):
        raise ApoeError(f"x must be a matrix or a batch of matrices, not {tuple(x.shape)}")
    in_dtype = _dtype(x, "x")
    if out is None:
        if beta != 0.0:
            raise ApoeError("beta without out")
        out = _torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out.shape != x.shape:
        raise ApoeError(f"out must be of shape {tuple(x.shape)}, not {tuple(out.shape)}")
    a = OrthogonalizeArgs()
    a.in_dtype, a.out_dtype = in_dtype, _dtype(out, "out")
    if products is None:
        products = "f16" if a.out_dtype == 2 else "f32"
    if products not in ("f16", "f32"):
        raise ApoeError(f'products must be "f16" or "f32", not {products!r}')
    a.products = 1 if products == "f16" else 0
    a.batch, (a.rows, a.cols) = (x.shape[0] if x.dim() == 3 else 1), x.shape[-2:]
    if x.numel() == 0:
        return out
    for t, name, row, mat in ((x, "x", "in_stride", "in_batch_stride"), (out, "out", "out_stride", "out_batch_stride")):
        setattr(a, row, _matrix(ctx, t if t.dim() == 2 else t[0], name))
        if t.dim() == 3 and t.shape[0] > 1:
            if t.stride(0) == 0:  # a matrix that is repeated: to the library zero would say that matrices follow one another
                raise ApoeError(f"the matrices of {name} overlap")
            setattr(a, mat, t.stride(0))
    a.in_, a.out, a.steps = x.data_ptr(), out.data_ptr(), steps
    a.a, a.b, a.c = coefs
    a.alpha, a.beta = alpha, beta
    _call(ctx, lib().apoe_orthogonalize, a)
    return out


def _residual_args(ctx, x, h, gate, scale, w_post, w_next, eps):
    a = GatedResidualArgs()
    a.dtype = _dtype(x, "x")
    a.x_stride = _matrix(ctx, x, "x")
    n, d = x.shape
    a.rows, a.dim, a.eps, a.x = n, d, eps, x.data_ptr()
    if h is not None:
        a.h_stride, a.h = _matrix(ctx, h, "h", (n, d), x.dtype), h.data_ptr()
    elif gate is not None or scale is not None or w_post is not None:
        raise ApoeError("gate, scale and w_post belong to a block: h is None")
    if gate is not None:
        if gate.dim() == 1:
            a.gate_kind, a.gate = 2, _vector(ctx, gate, "gate", d, (x.dtype,))
        else:
            a.gate_kind, a.gate_stride, a.gate = 1, _matrix(ctx, gate, "gate", (n, d), x.dtype), gate.data_ptr()
    for t, name in ((scale, "scale"), (w_post, "w_post"), (w_next, "w_next")):
        if t is not None:
            setattr(a, name, _vector(ctx, t, name, d, _FLOATS))
    return a


def gated_residual(ctx, x, h=None, gate=None, scale=None, w_post=None, w_next=None, eps=1e-6, want_u=True):
    """(y, u): y = x + scale * sigmoid(gate) * w_post * h / rms(h) and u = w_next * y / rms(y). gate: [n, d] or [d]; without h,
    y is x itself and u its norm."""
    a = _residual_args(ctx, x, h, gate, scale, w_post, w_next, eps)
    y = x if h is None else _torch.empty(x.shape, dtype=x.dtype, device=x.device)
    u = _torch.empty(x.shape, dtype=x.dtype, device=x.device) if want_u else None
    if x.numel() == 0:
        return y, u
    a.y = None if h is None else y.data_ptr()
    a.u = None if u is None else u.data_ptr()
    _call(ctx, lib().apoe_gated_residual, a)
    return y, u


def gated_residual_grad(ctx, x, h=None, gate=None, scale=None, w_post=None, w_next=None, eps=1e-6, grad_y=None, grad_u=None):
    """Gradients of gated_residual from those of y and u (either may be None): a dict of grad_x, and of grad_h, grad_gate,
    grad_scale, grad_w_post, grad_w_next for the inputs that are not None."""
    a = _residual_args(ctx, x, h, gate, scale, w_post, w_next, eps)
    n, d = x.shape
    if grad_y is None and grad_u is None:
        raise ApoeError("neither grad_y nor grad_u")
    for t, name in ((grad_y, "grad_y"), (grad_u, "grad_u")):
        if t is not None:
            setattr(a, name + "_stride", _matrix(ctx, t, name, (n, d), x.dtype))
            setattr(a, name, t.data_ptr())
    out = dict(grad_x=_torch.empty((n, d), dtype=x.dtype, device=x.device))
    if h is not None:
        out["grad_h"] = _torch.empty((n, d), dtype=x.dtype, device=x.device)
    if gate is not None:
        out["grad_gate"] = _torch.empty(gate.shape, dtype=x.dtype, device=x.device)
    for t, name in ((scale, "grad_scale"), (w_post, "grad_w_post"), (w_next, "grad_w_next")):
        if t is not None:
            out[name] = _torch.empty(d, dtype=_torch.float32, device=x.device)
    if x.numel() == 0:
        for v in out.values():
            v.zero_()
        return out
    for name, t in out.items():
        setattr(a, name, t.data_ptr())
    _call(ctx, lib().apoe_gated_residual_grad, a)
    return out


# ---- layers of an adapter, and their training ----

def _wanted(ctx, asked, name, shape, like):
    """The tensor that a gradient goes to: the caller's own (checked), or a new one where True is asked for. None: not wanted."""
    if asked is False or asked is None:
        return None
    if asked is True:
        return _torch.empty(shape, dtype=like.dtype, device=like.device)
    _matrix(ctx, asked, name, _torch.Size(shape), like.dtype)
    return asked


def _embed_args(ctx, table, idx, off, val, scale):
    a = EmbedArgs()
    a.dtype = _dtype(table, "table")
    a.table_stride = _matrix(ctx, table, "table")
    (a.n_table, a.dim), a.table = table.shape, table.data_ptr()
    a.idx = _vector(ctx, idx, "idx", None, _INTS)
    entries = idx.shape[0]
    a.n_entries, a.n_rows, a.scale = entries, entries, scale
    if off is not None:
        a.off = _vector(ctx, off, "off", None, _INTS)
        a.n_rows = off.shape[0] - 1
        if off.shape[0] == 0:
            raise ApoeError("off must have one number more than there are rows")
    if val is not None:
        a.val = _vector(ctx, val, "val", entries, _FLOATS)
    return a


def embed(ctx, table, idx, off=None, val=None, scale=1.0, base=None, out=None):
    """out[i] = base[i] + scale * the sum of val[e] * table[idx[e]] over the entries e of row i: off [m + 1], idx and val are the CSR of the
    rows' terms and weights (ones without val); without off entry i is row i's. Entries at or above the table's length count nothing. table, base and
    out have one type; out may be base itself."""
    a = _embed_args(ctx, table, idx, off, val, scale)
    shape = (a.n_rows, a.dim)
    if base is not None:
        a.base_stride, a.base = _matrix(ctx, base, "base", shape, table.dtype), base.data_ptr()
    if out is None:  # (like base where that is dense: half a microsecond less)
        out = table.new_empty(shape) if base is None or a.base_stride != a.dim else _torch.empty_like(base)
    else:
        a.out_stride = _matrix(ctx, out, "out", shape, table.dtype)
    a.out = out.data_ptr()
    if a.n_rows == 0 or a.dim == 0:
        return out
    _call(ctx, lib().apoe_embed, a)
    return out


def embed_grad(ctx, table, grad, idx, off=None, val=None, scale=1.0, grad_table=True, grad_val=False, accumulate=False):
    """Gradients of embed from that of out (which is base's own): a dict of grad_table (True, or a matrix like the table to write to, with
    accumulate to add to) and grad_val [entries]."""
    a = _embed_args(ctx, table, idx, off, val, scale)
    a.grad_stride, a.grad = _matrix(ctx, grad, "grad", _torch.Size((a.n_rows, a.dim)), table.dtype), grad.data_ptr()
    if accumulate and (grad_table is True or grad_table is False or grad_table is None):
        raise ApoeError("accumulate needs the grad_table that is added to")
    out = {}
    g = _wanted(ctx, grad_table, "grad_table", table.shape, table)
    if g is not None:
        a.grad_table_stride, a.grad_table, a.accumulate = _matrix(ctx, g, "grad_table"), g.data_ptr(), bool(accumulate)
        out["grad_table"] = g
    if grad_val:
        out["grad_val"] = _torch.empty(idx.shape[0], dtype=_torch.float32, device=table.device)
        a.grad_val = out["grad_val"].data_ptr()
    if not out:
        raise ApoeError("neither grad_table nor grad_val")
    if all(t.numel() == 0 for t in out.values()):
        return out
    if table.numel() == 0:  # no row that an entry could name
        out["grad_val"].zero_()
        return out
    if idx.numel() == 0 and a.grad_table is None:
        return out
    _call(ctx, lib().apoe_embed_grad, a)
    return out


def _norm_args(ctx, x, w, b, eps):
    a = LayerNormArgs()
    a.dtype = _dtype(x, "x")
    a.x_stride = _matrix(ctx, x, "x")
    (a.rows, d), a.eps, a.x = x.shape, eps, x.data_ptr()
    a.dim = d
    if w is not None:
        a.w = _vector(ctx, w, "w", d, _FLOATS)
    if b is not None:
        a.b = _vector(ctx, b, "b", d, _FLOATS)
    return a


def layer_norm(ctx, x, w=None, b=None, eps=1e-5, out=None):
    """w * (x - mean(x)) / sqrt(var(x) + eps) + b for every row of x [m, d]; w and b are float32. out may be x itself."""
    a = _norm_args(ctx, x, w, b, eps)
    if out is None:  # (like x where that is dense: half a microsecond less)
        out = _torch.empty_like(x) if a.x_stride == a.dim else x.new_empty(x.shape)
    else:
        a.y_stride = _matrix(ctx, out, "out", x.shape, x.dtype)
    a.y = out.data_ptr()
    if a.rows == 0 or a.dim == 0:
        return out
    _call(ctx, lib().apoe_layer_norm, a)
    return out


def layer_norm_grad(ctx, x, w=None, b=None, eps=1e-5, grad_y=None, grad_skip=None):
    """Gradients of layer_norm: a dict of grad_x (grad_skip, what x's gradient has by another way, is added to it), and of grad_w, grad_b for
    the vectors that are not None."""
    a = _norm_args(ctx, x, w, b, eps)
    if grad_y is None:
        raise ApoeError("grad_y is None")
    for t, name in ((grad_y, "grad_y"), (grad_skip, "grad_skip")):
        if t is not None:
            setattr(a, name + "_stride", _matrix(ctx, t, name, x.shape, x.dtype))
            setattr(a, name, t.data_ptr())
    out = dict(grad_x=_torch.empty(x.shape, dtype=x.dtype, device=x.device))
    for t, name in ((w, "grad_w"), (b, "grad_b")):
        if t is not None:
            out[name] = _torch.empty(a.dim, dtype=_torch.float32, device=x.device)
    if x.numel() == 0:
        for t in out.values():
            t.zero_()
        return out
    for name, t in out.items():
        setattr(a, name, t.data_ptr())
    _call(ctx, lib().apoe_layer_norm_grad, a)
    return out


ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


def _linear_args(ctx, x, w, act):
    a = LinearArgs()
    a.dtype = _dtype(x, "x")
    a.x_stride = _matrix(ctx, x, "x")
    a.w_stride = _matrix(ctx, w, "w", dtype=x.dtype)
    (m, k), (n, same) = x.shape, w.shape
    if same != k:
        raise ApoeError(f"w must have x's {k} columns, not {same}")
    if n == 0 or k == 0:
        raise ApoeError("w is empty")
    a.act = ACTIVATIONS.get(act, -1)
    if a.act > 3:
        raise ApoeError(f"act must be one of {', '.join(ACTIVATIONS)}, not {act!r}")
    a.rows, a.cols_in, a.cols_out, a.x, a.w = m, k, n, x.data_ptr(), w.data_ptr()
    return a


def linear(ctx, x, w, bias=None, act="none", residual=None, want_pre=False, out=None):
    """(y, pre): y = act(pre) + residual with pre = x w^T + bias, for x [m, k], w [n, k], bias [n] float32, residual [m, n]; act: "none", "relu",
    "gelu" or "silu". pre, which linear_grad needs where there is an activation, is None unless it is wanted."""
    a = _linear_args(ctx, x, w, act)
    n = a.cols_out
    shape = (a.rows, n)
    if bias is not None:
        a.bias = _vector(ctx, bias, "bias", n, _FLOATS)
    if residual is not None:
        a.residual_stride, a.residual = _matrix(ctx, residual, "residual", shape, x.dtype), residual.data_ptr()
    if out is None:
        out = x.new_empty(shape)
    else:
        a.y_stride = _matrix(ctx, out, "out", shape, x.dtype)
    a.y = out.data_ptr()
    pre = None
    if want_pre:
        pre = x.new_empty(shape)
        a.pre = pre.data_ptr()
    if shape[0] == 0:
        return out, pre
    _call(ctx, lib().apoe_linear, a)
    return out, pre


def linear_grad(ctx, x, w, grad_y, act="none", pre=None, grad_x=True, grad_w=True, grad_bias=True):
    """Gradients of linear from that of y (which is residual's own): a dict of grad_x, grad_w (True, or a matrix to write to) and grad_bias
    (float32). pre: what linear gave, where there is an activation."""
    a = _linear_args(ctx, x, w, act)
    shape = _torch.Size((a.rows, a.cols_out))
    a.grad_y_stride, a.grad_y = _matrix(ctx, grad_y, "grad_y", shape, x.dtype), grad_y.data_ptr()
    if a.act:
        if pre is None:
            raise ApoeError("the gradient of an activation needs pre")
        a.pre_stride, a.pre = _matrix(ctx, pre, "pre", shape, x.dtype), pre.data_ptr()
    out = {}
    for asked, name, t in ((grad_x, "grad_x", x), (grad_w, "grad_w", w)):
        g = _wanted(ctx, asked, name, t.shape, t)
        if g is not None:
            setattr(a, name + "_stride", _matrix(ctx, g, name))
            setattr(a, name, g.data_ptr())
            out[name] = g
    if grad_bias:
        out["grad_bias"] = _torch.empty(a.cols_out, dtype=_torch.float32, device=x.device)
        a.grad_bias = out["grad_bias"].data_ptr()
    if not out:
        raise ApoeError("nothing to compute")
    if x.shape[0] == 0:
        for t in out.values():
            t.zero_()
        return out
    _call(ctx, lib().apoe_linear_grad, a)
    return out


class AdamW:
    """AdamW over a list of float32 parameters (any shapes, contiguous; stepped in place).

    copies: for each parameter a float16 or bfloat16 tensor of its shape (or None) that gets the stepped values, rounded. bits: of the moments, 32 or 8
    (8: a code a value and a scale for every 256; rounded up or down by chance, which `seed` chooses). weight_decay: one number, or one for each
    parameter. state: what `state()` of an earlier object gave, used in place; by default the moments are zeros and no step has been taken.

    The moments of all parameters lie in one array each, parameter i from offsets[i] on (a multiple of 256)."""

    BLOCK = 256

    def __init__(self, ctx, params, copies=None, bits=32, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, seed=0, state=None):
        self.h = C.c_void_p()
        if _torch is None:
            _load_torch()
        self.ctx, self.bits, self.betas, self.eps, self.seed = ctx, bits, betas, eps, seed
        self.params = list(params)
        self.copies = [None] * len(self.params) if copies is None else list(copies)
        decay = list(weight_decay) if isinstance(weight_decay, (list, tuple)) else [weight_decay] * len(self.params)
        if bits not in (8, 32):
            raise ApoeError(f"moments have 8 or 32 bits, not {bits}")
        if len(self.copies) != len(self.params) or len(decay) != len(self.params):
            raise ApoeError("copies and weight_decay need one entry for each parameter")
        blocks, self.offsets = 0, []
        for p, c in zip(self.params, self.copies):
            self._checked(p, "a parameter", _FLOATS)
            if c is not None:
                self._checked(c, "a copy", (_torch.float16, _torch.bfloat16), p.shape)
            self.offsets.append(blocks * self.BLOCK)
            blocks += -(-p.numel() // self.BLOCK)
        n, dev = blocks * self.BLOCK, f"cuda:{ctx.device}"
        types = dict(m=_torch.float32, v=_torch.float32) if bits == 32 else dict(m=_torch.int8, v=_torch.uint8, m_scale=_torch.float32, v_scale=_torch.float32)
        if state is None:
            state = {k: _torch.zeros(blocks if k.endswith("scale") else n, dtype=t, device=dev) for k, t in types.items()}
        for k, t in types.items():
            if k not in state:
                raise ApoeError(f"state has no {k}")
            _vector(ctx, state[k], k, blocks if k.endswith("scale") else n, (t,))
        self._moments = {k: state[k] for k in types}
        self._taken, self._on_gpu = _torch.empty(1, dtype=_torch.int32, device=dev), False  # the last step's number, as the GPU took it
        self.t = int(state.get("t", 0))
        tensors = (AdamwTensor * len(self.params))()
        for a, p, c, d, at in zip(tensors, self.params, self.copies, decay, self.offsets):
            a.p, a.n, a.decay = p.data_ptr(), p.numel(), d
            for k, t in self._moments.items():
                setattr(a, k, t.data_ptr() + (at // self.BLOCK if k.endswith("scale") else at) * t.element_size())
            if c is not None:
                a.copy, a.copy_dtype = c.data_ptr(), _DTYPES[c.dtype]
        _check(lib().apoe_adamw_create(ctx.h, C.c_uint32(len(self.params)), tensors, C.c_uint32(bits), C.c_uint32(seed & 0xFFFFFFFF), C.byref(self.h)))
        self._grads, self._types = (C.c_void_p * len(self.params))(), (C.c_uint32 * len(self.params))()
        self._sizes = [p.numel() for p in self.params]

    def _checked(self, t, name, dtypes, shape=None):
        _on_gpu(self.ctx, t, name)
        if t.dtype not in dtypes or not t.is_contiguous() or (shape is not None and t.shape != shape):
            raise ApoeError(f"{name} must be a contiguous tensor of {' or '.join(str(d) for d in dtypes)}{'' if shape is None else f' of shape {tuple(shape)}'}")

    @property
    def t(self):
        """The number of steps taken. (After steps whose number is a tensor it is asked of the GPU, which is waited for.)"""
        if self._on_gpu:
            if _torch.cuda.is_current_stream_capturing():
                raise ApoeError("the number of steps taken is the GPU's after steps whose number was a tensor: during a capture give t")
            _torch.cuda.synchronize(self.ctx.device)
            return int(self._taken)
        return self._t

    @t.setter
    def t(self, t):
        self._t = t
        self._taken.fill_(t)

    def step(self, grads, lr, grad_scale=1.0, t=None):
        """One step with the parameters' gradients (None: that parameter and its moments stay as they are), which count times grad_scale. lr may be a
        float32 tensor of one number on the GPU, and t, the number of the step, an int32 one: a captured step reads both when it
        is replayed (the program counts t up; without it the object counts on from the last step that was taken)."""
        if not (self.h and self.ctx.h):
            raise ApoeError("the object or its context has been closed")
        if len(grads) != len(self.params):
            raise ApoeError(f"{len(grads)} gradients for {len(self.params)} parameters")
        a = AdamwStepArgs()
        for i, g in enumerate(grads):
            if g is None:
                self._grads[i] = None
                continue
            if g.get_device() != self.ctx.device or g.numel() != self._sizes[i] or not g.is_contiguous():
                raise ApoeError(f"gradient {i} must be a contiguous tensor of {self._sizes[i]} values on GPU {self.ctx.device}, the context's")
            self._types[i] = _dtype(g, "a gradient")
            self._grads[i] = g.data_ptr()
        a.grads, a.grad_dtypes = C.addressof(self._grads), C.addressof(self._types)
        if isinstance(lr, _torch.Tensor):
            a.lr_dev = _vector(self.ctx, lr.reshape(-1), "lr", 1, _FLOATS)
        else:
            a.lr = lr
        a.beta1, a.beta2 = self.betas
        a.eps, a.grad_scale, a.step_taken = self.eps, grad_scale, self._taken.data_ptr()
        if t is not None:
            a.step_dev = _vector(self.ctx, t.reshape(-1), "t", 1, _INTS)
        else:
            a.step = self.t + 1
        _ordered(self.ctx, lambda: lib().apoe_adamw_step(self.h, C.byref(a)))
        if t is None:
            self._t = a.step
        else:
            self._on_gpu = True  # from now on: a captured step may be replayed at any time

    def moments(self):
        """(m, v) as float32, laid out like the moments themselves: those themselves where they have 32 bits."""
        m = self._moments
        if self.bits == 32:
            return m["m"], m["v"]
        out = [_torch.empty(t.shape, dtype=_torch.float32, device=t.device) for t in (m["m"], m["v"])]
        pointers = [C.c_void_p(t.data_ptr()) for t in (m["m"], m["m_scale"], m["v"], m["v_scale"], *out)]
        _ordered(self.ctx, lambda: lib().apoe_adamw_moments(self.ctx.h, C.c_uint64(m["m"].numel()), *pointers))
        return tuple(out)

    def state(self):
        """What another object over the same parameters goes on from (the arrays themselves, not copies)."""
        return dict(self._moments, t=self.t)

    def close(self):
        if self.h:
            lib().apoe_adamw_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
