"""Host-side mirror of the reference's lns_cuda::kernel_set
(lns-backend/cuda/lns-cuda-kernels.h:85-139) over the C ABI of
include/lnsb200.h.

One KernelSet per (summation-mode build, format), like the reference's
xlns16_kernels() / xlns32_kernels().  Tensors are torch CUDA tensors used
purely as device memory: uint16 (xlns16 codes), int32 (xlns32 codes, same
bits as uint32) or float32.  Every call launches asynchronously on the
current torch stream (or the given one) and raises LnsbError on failure --
there is no CPU fallback.
"""
import ctypes

from . import _lib
from ._lib import MODES, XLNS16, XLNS32, LnsbError, MulMatArgs, Shape4, SoftMaxArgs  # noqa: F401

__all__ = ["KernelSet", "MODES", "XLNS16", "XLNS32", "LnsbError", "MulMatArgs", "SoftMaxArgs", "Shape4",
           "kernels", "monte_get_state", "monte_set_state", "monte_reserve"]


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(stream):
    import torch
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _shape4(shape):
    ne = list(shape) + [1] * (4 - len(shape))
    return Shape4((ctypes.c_int64 * 4)(*ne))


class KernelSet:
    """kernel_set for one format of one summation-mode build."""

    def __init__(self, fmt=XLNS16, mode="base"):
        if fmt not in (XLNS16, XLNS32):
            raise ValueError("format must be 16 or 32")
        self.fmt = fmt
        self.mode = mode
        self.lib = _lib.load(mode)

    # ---- identity (kernel_set::format_name ... monte_impl) ----
    def format_name(self):
        return self.lib.lnsb_format_name(self.fmt).decode()

    def value_size(self):
        return self.lib.lnsb_value_size(self.fmt)

    def sum_mode(self):
        r = self.lib.lnsb_sum_mode(self.fmt)
        return r.decode() if r else None

    def monte_impl(self):
        r = self.lib.lnsb_monte_impl(self.fmt)
        return r.decode() if r else None

    def description(self):
        return self.lib.lnsb_description(self.fmt).decode()

    # ---- draw accounting ----
    def mul_mat_draws(self, K, M, N, ne02=1, ne03=1, ne12=1, ne13=1):
        a = MulMatArgs(None, None, None, K, M, N, ne02, ne03, ne12, ne13, 0)
        return self.lib.lnsb_mul_mat_draws(self.fmt, ctypes.byref(a))

    def soft_max_draws(self, ncols, nrows):
        return self.lib.lnsb_soft_max_draws(self.fmt, ncols, nrows)

    def rms_norm_draws(self, ncols, nrows):
        return self.lib.lnsb_rms_norm_draws(self.fmt, ncols, nrows)

    # ---- tables / conversions ----
    def upload_tables(self):
        _lib.check(self.lib, "lnsb_upload_tables", self.lib.lnsb_upload_tables(self.fmt))

    def add_latency(self, kind, lanes=32, steps=4096):
        """SM cycles of one dependent LNS addition (lnsb_add_latency): kind 0 the
        key-form xlns16 addition of the latency mul_mat kernels, 1 / 2 the
        non-negative xlns16 / xlns32 additions of the normalisers, 3 the
        general xlns32 addition of the latency mat-vecs (sum32, xlns32)"""
        import torch
        out = torch.zeros(2, dtype=torch.int64, device="cuda")
        _lib.check(self.lib, "lnsb_add_latency", self.lib.lnsb_add_latency(kind, lanes, steps, _ptr(out), None))
        torch.cuda.synchronize()
        return out[0].item() / (steps - 1)

    def to_lns(self, src, dst, stream=None):
        _lib.check(self.lib, "lnsb_to_lns", self.lib.lnsb_to_lns(self.fmt, _ptr(src), _ptr(dst), src.numel(), _stream(stream)))

    def to_lns_transposed(self, src, dst, rows, cols, dst_ld, stream=None):
        _lib.check(self.lib, "lnsb_to_lns_transposed",
                   self.lib.lnsb_to_lns_transposed(self.fmt, _ptr(src), _ptr(dst), rows, cols, dst_ld, _stream(stream)))

    def to_f32(self, src, dst, stream=None):
        _lib.check(self.lib, "lnsb_to_f32", self.lib.lnsb_to_f32(self.fmt, _ptr(src), _ptr(dst), src.numel(), _stream(stream)))

    # ---- the hot path ----
    def _mm_args(self, w, x, dst, K, M, N, slices, monte_seed):
        ne02, ne03, ne12, ne13 = slices
        return MulMatArgs(w.data_ptr(), x.data_ptr(), dst.data_ptr() if dst is not None else None,
                          K, M, N, ne02, ne03, ne12, ne13, monte_seed)

    def mul_mat(self, w, x, dst, K, M, N, slices=(1, 1, 1, 1), monte_seed=7, stream=None):
        """dst (F32, [slices][N][M]) = W^T x; w k-major [K][M] per weight slice, x [N][K]."""
        a = self._mm_args(w, x, dst, K, M, N, slices, monte_seed)
        _lib.check(self.lib, "lnsb_mul_mat", self.lib.lnsb_mul_mat(self.fmt, ctypes.byref(a), _stream(stream)))

    def mul_mat_xf32(self, w, x_f32, x_work, dst, K, M, N, slices=(1, 1, 1, 1), monte_seed=7, stream=None):
        """the MUL_MAT op over F32 activations (lnsb_mul_mat_xf32): x_f32 [N][K] floats, converted as
        the kernel stages them or into x_work (N*K codes) first; dst F32 as mul_mat"""
        a = self._mm_args(w, x_f32, dst, K, M, N, slices, monte_seed)
        _lib.check(self.lib, "lnsb_mul_mat_xf32",
                   self.lib.lnsb_mul_mat_xf32(self.fmt, ctypes.byref(a), _ptr(x_work), _stream(stream)))

    def mul_mat_lns(self, w, x, dst, K, M, N, slices=(1, 1, 1, 1), monte_seed=7, stream=None):
        """as mul_mat with LNS codes out"""
        a = self._mm_args(w, x, None, K, M, N, slices, monte_seed)
        _lib.check(self.lib, "lnsb_mul_mat_lns", self.lib.lnsb_mul_mat_lns(self.fmt, ctypes.byref(a), _ptr(dst), _stream(stream)))

    def attn_decode(self, q, k_cache, v_cache, kv_ld, nkv, n_head, n_head_kv, head_dim, scale, dst, monte_seed=7,
                    stream=None, dst_lns=None):
        """one decode step's attention (lnsb_attn_decode): q F32 [n_head][head_dim], caches F16
        [nkv][kv_ld], dst F32 [n_head][head_dim] (or None), dst_lns its codes (optional)"""
        a = _lib.AttnDecodeArgs(_ptr(q), _ptr(k_cache), _ptr(v_cache), kv_ld, nkv, n_head, n_head_kv, head_dim, scale,
                                _ptr(dst) if dst is not None else None, monte_seed,
                                _ptr(dst_lns) if dst_lns is not None else None)
        _lib.check(self.lib, "lnsb_attn_decode", self.lib.lnsb_attn_decode(self.fmt, ctypes.byref(a), _stream(stream)))

    def norm_block(self, src, dst_lns, ncols, nrows, eps, residual=None, x_out=None, weight=None, monte_seed=7,
                   stream=None):
        """lnsb_norm_block: [residual add,] rms_norm, [times weight,] to_lns"""
        opt = lambda t: _ptr(t) if t is not None else None
        a = _lib.NormBlockArgs(_ptr(src), opt(residual), opt(x_out), opt(weight), _ptr(dst_lns), ncols, nrows, eps,
                               monte_seed)
        _lib.check(self.lib, "lnsb_norm_block", self.lib.lnsb_norm_block(self.fmt, ctypes.byref(a), _stream(stream)))

    def glu_lns(self, gate, up, gate_stride, up_stride, dst_lns, ncols, nrows, op="swiglu", stream=None):
        _lib.check(self.lib, "lnsb_glu_lns", self.lib.lnsb_glu_lns(self.fmt, 0 if op == "swiglu" else 1, _ptr(gate),
                                                                   _ptr(up), gate_stride, up_stride, _ptr(dst_lns),
                                                                   ncols, nrows, _stream(stream)))

    def rope_qkv(self, qkv, ld, cos_sin, n_dims, n_head, n_head_kv, head_dim, n_tokens, q_out, k_cache, v_cache, kv_ld,
                 neox=False, stream=None):
        a = _lib.RopeQkvArgs(_ptr(qkv), ld, _ptr(cos_sin), n_dims, 1 if neox else 0, n_head, n_head_kv, head_dim,
                             n_tokens, _ptr(q_out), _ptr(k_cache), _ptr(v_cache), kv_ld)
        _lib.check(self.lib, "lnsb_rope_qkv", self.lib.lnsb_rope_qkv(self.fmt, ctypes.byref(a), _stream(stream)))

    def attn_decode_max_keys(self, head_dim):
        return self.lib.lnsb_attn_decode_max_keys(self.fmt, head_dim)

    def type_row_bytes(self, type, cols):
        return self.lib.lnsb_type_row_bytes(_lib.TYPES.get(type, type), cols)

    def to_lns_transposed_typed(self, type, src, dst, rows, cols, dst_ld, stream=None):
        """dst[c * dst_ld + r] = lns(value c of row r); src rows in a ggml storage type (name or id)"""
        _lib.check(self.lib, "lnsb_to_lns_transposed_typed",
                   self.lib.lnsb_to_lns_transposed_typed(self.fmt, _lib.TYPES.get(type, type), _ptr(src), _ptr(dst),
                                                         rows, cols, dst_ld, _stream(stream)))

    def dequantize(self, type, src, dst, rows, cols, stream=None):
        _lib.check(self.lib, "lnsb_dequantize",
                   self.lib.lnsb_dequantize(_lib.TYPES.get(type, type), _ptr(src), _ptr(dst), rows, cols, _stream(stream)))

    def mul_mat_lns_peers(self, w, x, ptrs_dev, n_peers, ld, offset, K, M, N, slices=(1, 1, 1, 1), monte_seed=7,
                          stream=None):
        """mul_mat with the output-row all-gather fused into the store: codes
        into every peer buffer (ptrs_dev: device address of an array of
        n_peers pointers) at [N][ld] columns [offset, offset + M)"""
        a = self._mm_args(w, x, None, K, M, N, slices, monte_seed)
        p = _lib.PeerOut(ptrs_dev, n_peers, ld, offset)
        _lib.check(self.lib, "lnsb_mul_mat_lns_peers",
                   self.lib.lnsb_mul_mat_lns_peers(self.fmt, ctypes.byref(a), ctypes.byref(p), _stream(stream)))

    def _mmid_args(self, w, x, ids, dst, K, M, n_expert, ne11, n_used, n_tokens, monte_seed):
        return _lib.MulMatIdArgs(w.data_ptr(), x.data_ptr(), ids.data_ptr(), dst.data_ptr() if dst is not None else None,
                                 K, M, n_expert, ne11, n_used, n_tokens, n_used, monte_seed)

    def mul_mat_id(self, w, x, ids, dst, K, M, n_expert, ne11, n_used, n_tokens, monte_seed=7, stream=None):
        """MUL_MAT_ID: dst (F32, [n_tokens][n_used][M]); w k-major [n_expert][K][M],
        x [n_tokens][ne11][K], ids int32 [n_tokens][n_used] on the device."""
        a = self._mmid_args(w, x, ids, dst, K, M, n_expert, ne11, n_used, n_tokens, monte_seed)
        _lib.check(self.lib, "lnsb_mul_mat_id", self.lib.lnsb_mul_mat_id(self.fmt, ctypes.byref(a), _stream(stream)))

    def mul_mat_id_lns(self, w, x, ids, dst, K, M, n_expert, ne11, n_used, n_tokens, monte_seed=7, stream=None):
        a = self._mmid_args(w, x, ids, None, K, M, n_expert, ne11, n_used, n_tokens, monte_seed)
        _lib.check(self.lib, "lnsb_mul_mat_id_lns",
                   self.lib.lnsb_mul_mat_id_lns(self.fmt, ctypes.byref(a), _ptr(dst), _stream(stream)))

    def mul_mat_id_draws(self, K, M, n_used, n_tokens):
        a = _lib.MulMatIdArgs(None, None, None, None, K, M, 1, 1, n_used, n_tokens, n_used, 0)
        return self.lib.lnsb_mul_mat_id_draws(self.fmt, ctypes.byref(a))

    def mul_mat_id_bad_ids(self):
        """out-of-range ids met on the current device since the last call"""
        c = ctypes.c_int64()
        _lib.check(self.lib, "lnsb_mul_mat_id_bad_ids", self.lib.lnsb_mul_mat_id_bad_ids(ctypes.byref(c)))
        return c.value

    def soft_max(self, src, shape, dst, work, mask=None, mask_shape=None, scale=1.0, monte_seed=7, stream=None):
        a = SoftMaxArgs(src.data_ptr(), _shape4(shape), mask.data_ptr() if mask is not None else None,
                        _shape4(mask_shape or (1, 1, 1, 1)), scale, dst.data_ptr(), work.data_ptr(), monte_seed)
        _lib.check(self.lib, "lnsb_soft_max", self.lib.lnsb_soft_max(self.fmt, ctypes.byref(a), _stream(stream)))

    def soft_max_lns(self, src, shape, dst, work, mask=None, mask_shape=None, scale_code=0x4000, monte_seed=7, stream=None):
        ne = (ctypes.c_int64 * 4)(*(list(shape) + [1] * (4 - len(shape))))
        mne = (ctypes.c_int64 * 4)(*(list(mask_shape) + [1] * (4 - len(mask_shape)))) if mask is not None else None
        _lib.check(self.lib, "lnsb_soft_max_lns",
                   self.lib.lnsb_soft_max_lns(self.fmt, _ptr(src), ne, _ptr(mask), mne, scale_code, _ptr(dst),
                                              _ptr(work), monte_seed, _stream(stream)))

    def rms_norm(self, src, dst, ncols, nrows, eps, monte_seed=7, stream=None):
        _lib.check(self.lib, "lnsb_rms_norm",
                   self.lib.lnsb_rms_norm(self.fmt, _ptr(src), _ptr(dst), ncols, nrows, eps, monte_seed, _stream(stream)))

    def rms_norm_lns(self, src, dst, ncols, nrows, eps, monte_seed=7, stream=None):
        _lib.check(self.lib, "lnsb_rms_norm_lns",
                   self.lib.lnsb_rms_norm_lns(self.fmt, _ptr(src), _ptr(dst), ncols, nrows, eps, monte_seed, _stream(stream)))


    # ---- elementwise ops of the model graph (F32 in and out) ----
    BINARY = {"add": 0, "mul": 1, "div": 2}
    UNARY = {"silu": 0, "gelu": 1, "relu": 2, "tanh": 3}

    def binary(self, op, a, a_shape, b, b_shape, dst, stream=None):
        """dst = a op b, b repeated to a's shape; shapes ggml order (ne0 innermost)"""
        ane, bne = _shape4(a_shape).ne, _shape4(b_shape).ne
        _lib.check(self.lib, "lnsb_binary", self.lib.lnsb_binary(self.fmt, self.BINARY[op], _ptr(a), ane, _ptr(b), bne,
                                                                 _ptr(dst), _stream(stream)))

    def scale(self, src, dst, n, s, b=0.0, stream=None):
        _lib.check(self.lib, "lnsb_scale", self.lib.lnsb_scale(self.fmt, _ptr(src), _ptr(dst), n, s, b, _stream(stream)))

    def unary(self, op, src, dst, n, stream=None):
        _lib.check(self.lib, "lnsb_unary", self.lib.lnsb_unary(self.fmt, self.UNARY[op], _ptr(src), _ptr(dst), n,
                                                               _stream(stream)))

    def glu(self, gate, up, gate_stride, up_stride, dst, ncols, nrows, op="swiglu", stream=None):
        _lib.check(self.lib, "lnsb_glu", self.lib.lnsb_glu(self.fmt, 0 if op == "swiglu" else 1, _ptr(gate), _ptr(up),
                                                           gate_stride, up_stride, _ptr(dst), ncols, nrows, _stream(stream)))

    def rope(self, src, shape, cos_sin, n_dims, dst, neox=False, stream=None):
        a = _lib.RopeArgs(_ptr(src), _shape4(shape), _ptr(cos_sin), n_dims, 1 if neox else 0, _ptr(dst))
        _lib.check(self.lib, "lnsb_rope", self.lib.lnsb_rope(self.fmt, ctypes.byref(a), _stream(stream)))

    def f32_to_f16(self, src, dst, n, stream=None):
        _lib.check(self.lib, "lnsb_f32_to_f16", self.lib.lnsb_f32_to_f16(_ptr(src), _ptr(dst), n, _stream(stream)))

    def f16_to_f32(self, src, dst, n, stream=None):
        _lib.check(self.lib, "lnsb_f16_to_f32", self.lib.lnsb_f16_to_f32(_ptr(src), _ptr(dst), n, _stream(stream)))


    # ---- serving many sequences from a paged KV cache (no LNS: any format, any mode).  A token's
    # latency is a few microseconds of GPU time, so these bindings keep to few Python steps ----
    def paged_append(self, k, v, k_cache, v_cache, page_table, q_start, kv_len, max_kv, q=None, q_out=None, cos_sin=None,
                     neox=False, stream=None):
        """lnsb_paged_append: k, v [n_tokens][n_head_kv][head_dim] (F32, F16 or BF16; token rows any distance apart) into
        the caches [n_pages][page_size][n_head_kv][head_dim] (F16 or BF16; any strides, heads contiguous), k turned by
        cos_sin [rows][n_dims / 2][2] (F32; None: not turned); q [n_tokens][n_head][head_dim] turned into q_out (of the
        caches' type).  The plan: page_table [n_seqs][pages], q_start [n_seqs + 1], kv_len [n_seqs], int32 on the device"""
        T, n_head_kv, D = k.shape
        kv = _paged_kv(k_cache, v_cache, page_table, q_start, kv_len, max_kv, T)
        ks, vs, ty = k.stride(), v.stride(), k.dtype
        if not (v.shape == k.shape and v.dtype is ty and ty in _type_ids and kv[15] == n_head_kv and kv[16] == D
                and _rows_ok(ks, n_head_kv, D) and _rows_ok(vs, n_head_kv, D)):
            raise ValueError("k and v must be [n_tokens][n_head_kv][head_dim] of one type (F32, F16, BF16), heads contiguous")
        dev = k_cache.get_device()
        if not dev == k.get_device() == v.get_device():
            raise ValueError(_elsewhere)
        cs = qp = op = None
        n_dims = n_head = q_ld = o_ld = 0
        if cos_sin is not None:
            rows, half, two = cos_sin.shape
            if not (cos_sin.dtype is _f32 and two == 2 and rows >= max_kv and cos_sin.is_contiguous()):
                raise ValueError("cos_sin must be contiguous F32 [rows >= max_kv][n_dims / 2][2]")
            if cos_sin.get_device() != dev:
                raise ValueError(_elsewhere)
            n_dims, cs = 2 * half, cos_sin.data_ptr() if half else None
        if q is not None:
            n, n_head, d = q.shape
            qs, qos = q.stride(), q_out.stride() if q_out is not None else ()
            if not (q_out is not None and q_out.shape == q.shape and q.dtype is ty and q_out.dtype is k_cache.dtype and n == T
                    and d == D and _rows_ok(qs, n_head, D) and _rows_ok(qos, n_head, D)):
                raise ValueError("q must be [n_tokens][n_head][head_dim] of k's type, q_out the same of the caches' type")
            if not dev == q.get_device() == q_out.get_device():
                raise ValueError(_elsewhere)
            q_ld, o_ld, qp, op = _ld(qs, T, n_head, D), _ld(qos, T, n_head, D), q.data_ptr(), q_out.data_ptr()
        a = _lib.PagedAppendArgs(*kv, k.data_ptr(), v.data_ptr(), qp, op, cs, _ld(ks, T, n_head_kv, D), _ld(vs, T, n_head_kv, D),
                                 q_ld, o_ld, _type_ids[ty], n_head, n_dims, 1 if neox else 0)
        st = self.lib.lnsb_paged_append(ctypes.byref(a), _raw_stream(stream))
        if st:
            _lib.check(self.lib, "lnsb_paged_append", st)

    def paged_attn_work(self, device=None):
        """a workspace for paged_attn on one stream (zeroed, as its first use wants it)"""
        import torch
        return torch.zeros(self.lib.lnsb_paged_attn_work_bytes(), dtype=torch.uint8, device=device or "cuda")

    def paged_attn(self, q, k_cache, v_cache, page_table, q_start, kv_len, max_q, max_kv, dst, work, scale=None, window=0,
                   stream=None):
        """lnsb_paged_attn: q, dst [n_tokens][n_head][head_dim] of the caches' type; the plan as in paged_append; scale
        None: 1 / sqrt(head_dim); window 0: every earlier row is visible"""
        T, n_head, D = q.shape
        kv = _paged_kv(k_cache, v_cache, page_table, q_start, kv_len, max_kv, T)
        qs, ds, ty = q.stride(), dst.stride(), k_cache.dtype
        if not (q.dtype is ty and dst.dtype is ty and dst.shape == q.shape and kv[16] == D and _rows_ok(qs, n_head, D)
                and _rows_ok(ds, n_head, D)):
            raise ValueError("q and dst must be [n_tokens][n_head][head_dim] of the caches' type, heads contiguous")
        if not k_cache.get_device() == q.get_device() == dst.get_device() == work.get_device():
            raise ValueError(_elsewhere)
        a = _lib.PagedAttnArgs(*kv, q.data_ptr(), dst.data_ptr(), work.data_ptr(), work.nbytes, _ld(qs, T, n_head, D),
                               _ld(ds, T, n_head, D), max_q, window, n_head, D ** -0.5 if scale is None else scale)
        st = self.lib.lnsb_paged_attn(ctypes.byref(a), _raw_stream(stream))
        if st:
            _lib.check(self.lib, "lnsb_paged_attn", st)

    def paged_attn_timeouts(self, work):
        """waits that ran out in the calls that used this workspace (read on the current stream): if there are any, those
        calls' outputs are invalid, and the workspace has to be zeroed"""
        import torch
        n = self.lib.lnsb_paged_attn_work_bytes()
        return work.view(torch.uint8)[n - 8:n].view(torch.int64).item()

    def paged_attn_wait_limit(self, cycles):
        """the most SM clock cycles that a wait inside paged_attn may take (lnsb_paged_attn_wait_limit)"""
        _lib.check(self.lib, "lnsb_paged_attn_wait_limit", self.lib.lnsb_paged_attn_wait_limit(cycles))

    def paged_errors(self):
        """(page ids outside the cache, waits that ran out) since the last call, on the current device"""
        b, t = ctypes.c_int64(), ctypes.c_int64()
        _lib.check(self.lib, "lnsb_paged_errors", self.lib.lnsb_paged_errors(ctypes.byref(b), ctypes.byref(t)))
        return b.value, t.value

    def sample(self, logits, u, token, prob=None, temperature=None, top_k=None, top_p=None, min_p=None, stream=None):
        """lnsb_sample: the next token of every row of logits [n_rows][n_vocab] (F32, F16 or BF16; rows any distance
        apart) from one number u [n_rows] in [0, 1); token int32 [n_rows], prob F32 [n_rows] or None; temperature,
        top_p, min_p F32 [n_rows] and top_k int32 [n_rows], each or None"""
        R, V = logits.shape
        if not _type_ids:
            _load_types()
        ld, step = logits.stride()
        if not ((step == 1 or V == 1) and logits.dtype in _type_ids):
            raise ValueError("logits must be F32, F16 or BF16 with contiguous rows")
        d = logits.get_device()
        a = _lib.SampleArgs(logits.data_ptr(), _row_ptr(temperature, _f32, R, d), _row_ptr(top_k, _i32, R, d),
                            _row_ptr(top_p, _f32, R, d), _row_ptr(min_p, _f32, R, d), _row_ptr(u, _f32, R, d),
                            _row_ptr(token, _i32, R, d), _row_ptr(prob, _f32, R, d), ld if R > 1 else V, R, V,
                            _type_ids[logits.dtype])
        if d < 0 or d != _current_device():
            raise ValueError(_elsewhere)
        st = self.lib.lnsb_sample(ctypes.byref(a), _raw_stream(stream))
        if st:
            _lib.check(self.lib, "lnsb_sample", st)


# torch's types, looked up at the first use (the module itself does not import torch)
_type_ids = {}
_f32 = _i32 = _current_stream = _current_device = None


def _load_types():
    global _f32, _i32, _current_stream, _current_device
    import torch
    try:                                # the same handle without a Stream object: 0.2 us, not 3
        raw, device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
        _current_stream, _current_device = lambda: raw(device()), device
    except AttributeError:
        _current_device = torch.cuda.current_device
        _current_stream = lambda: torch.cuda.current_stream().cuda_stream  # noqa: E731
    _f32, _i32 = torch.float32, torch.int32
    _type_ids.update({_f32: _lib.TYPES["f32"], torch.float16: _lib.TYPES["f16"], torch.bfloat16: _lib.TYPES["bf16"]})


def _raw_stream(stream):
    """the given or the current stream's cudaStream_t"""
    return stream.cuda_stream if stream is not None else _current_stream()


def _rows_ok(st, heads, D):
    """strides of [tokens][heads][D] whose rows are contiguous"""
    return st[2] == 1 and (st[1] == D or heads == 1)


def _ld(st, tokens, heads, D):
    """elements between token rows; the stride of a single one may be anything"""
    return st[0] if tokens > 1 else heads * D


_elsewhere = "every tensor must be on the current CUDA device"


def _row_ptr(t, dtype, rows, dev):
    if t is None:
        return None
    if not (t.dtype is dtype and t.numel() == rows and t.is_contiguous()):
        raise ValueError("u, prob, temperature, top_p, min_p must be F32 [n_rows], token and top_k int32 [n_rows]")
    if t.get_device() != dev:
        raise ValueError(_elsewhere)
    return t.data_ptr()


def _paged_kv(k_cache, v_cache, page_table, q_start, kv_len, max_kv, n_tokens):
    """the fields of lnsb_paged_kv"""
    if not _type_ids:
        _load_types()
    n_pages, page_size, n_head_kv, head_dim = shape = k_cache.shape
    st, ty = k_cache.stride(), k_cache.dtype
    if not (v_cache.dtype is ty and ty in _type_ids and v_cache.shape == shape and v_cache.stride() == st and st[3] == 1):
        raise ValueError("k_cache and v_cache must be [n_pages][page_size][n_head_kv][head_dim] of one type, with the same "
                         "strides and contiguous heads")
    n_seqs, table_ld = page_table.shape
    if not (page_table.dtype is _i32 and q_start.dtype is _i32 and kv_len.dtype is _i32 and q_start.numel() == n_seqs + 1
            and kv_len.numel() == n_seqs and page_table.is_contiguous() and q_start.is_contiguous() and kv_len.is_contiguous()):
        raise ValueError("page_table [n_seqs][pages], q_start [n_seqs + 1] and kv_len [n_seqs] must be contiguous int32")
    dev = k_cache.get_device()
    if not (0 <= dev == v_cache.get_device() == page_table.get_device() == q_start.get_device() == kv_len.get_device()
            and dev == _current_device()):
        raise ValueError(_elsewhere)
    return (k_cache.data_ptr(), v_cache.data_ptr(), st[0], st[1], st[2], page_table.data_ptr(), q_start.data_ptr(),
            kv_len.data_ptr(), table_ld, n_pages, n_tokens, max_kv, n_seqs, _type_ids[ty], page_size, n_head_kv, head_dim, 0)


def kernels(fmt=XLNS16, mode="base"):
    return KernelSet(fmt, mode)


# ---- Monte state (ggml-lns.h:13-24): process-wide, per monte build ----
def monte_get_state(mode="monte"):
    lib = _lib.load(mode)
    s = ctypes.c_uint16()
    _lib.check(lib, "lnsb_monte_get_state", lib.lnsb_monte_get_state(ctypes.byref(s)))
    return s.value


def monte_set_state(state, mode="monte"):
    lib = _lib.load(mode)
    _lib.check(lib, "lnsb_monte_set_state", lib.lnsb_monte_set_state(state))


def monte_reserve(draws, mode="monte"):
    lib = _lib.load(mode)
    s = ctypes.c_uint16()
    _lib.check(lib, "lnsb_monte_reserve", lib.lnsb_monte_reserve(draws, ctypes.byref(s)))
    return s.value


class WeightCache:
    """lnsb_weight_cache_*: weights converted to LNS once per (data pointer,
    type, rows, cols) and kept on the device within a byte budget
    (budget < 0: GGML_LNS_CUDA_CACHE_MB, else free memory less 1 GiB)."""

    def __init__(self, ks, budget=-1):
        self.ks = ks
        self.lib = ks.lib
        self.h = self.lib.lnsb_weight_cache_create(ks.fmt, budget)
        if not self.h:
            raise LnsbError(self.lib, "lnsb_weight_cache_create", -1)

    def get(self, src, type, rows, cols, scratch=None, stream=None):
        """device address of the k-major LNS image of `src` (a torch tensor
        on the device, or a numpy array / address in host memory)"""
        out = ctypes.c_void_p()
        _lib.check(self.lib, "lnsb_weight_cache_get",
                   self.lib.lnsb_weight_cache_get(self.h, _addr(src), _lib.TYPES.get(type, type), rows, cols,
                                                  _ptr(scratch) if scratch is not None else None, ctypes.byref(out),
                                                  _stream(stream)))
        return out.value

    def stats(self):
        e, u, b = ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int64()
        _lib.check(self.lib, "lnsb_weight_cache_stats",
                   self.lib.lnsb_weight_cache_stats(self.h, ctypes.byref(e), ctypes.byref(u), ctypes.byref(b)))
        return {"entries": e.value, "used": u.value, "budget": b.value}

    def close(self):
        if self.h:
            self.lib.lnsb_weight_cache_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _addr(obj):
    """device or host address of a torch tensor, a numpy array or an int"""
    if hasattr(obj, "data_ptr"):
        return obj.data_ptr()
    if hasattr(obj, "ctypes"):
        return obj.ctypes.data
    return int(obj)
