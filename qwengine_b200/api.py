"""ctypes binding of the C ABI (include/q38b200.h) for torch CUDA tensors.

Mirrors the reference's CUDA-side interface for this path (src/cuda/gemv.cuh:14-37,
src/cuda/prefill.cuh:17-28): weights are uint8 tensors holding GGUF blocks row by row, outputs are
``y[c, r]`` (column-major in the reference's sense: column c at ``y + c * y_ld``).
"""
import ctypes as C
import os
import struct

import torch

from . import formats as F

_HERE = os.path.dirname(os.path.abspath(__file__))
_LIB = None

OUT_F32, OUT_F16, OUT_BF16 = 0, 1, 2
_OUT_DTYPES = {OUT_F32: torch.float32, OUT_F16: torch.float16, OUT_BF16: torch.bfloat16}
_OUT_KINDS = {d: k for k, d in _OUT_DTYPES.items()}


class Q38BError(RuntimeError):
    def __init__(self, status, what):
        self.status = status
        super().__init__(f"{what}: {status_string(status)} ({status})")


def library_path():
    return os.path.join(_HERE, "libq38b200.so")


def load_library():
    """Loads libq38b200.so; raises if it has not been built (there is no fallback path)."""
    global _LIB
    if _LIB is not None:
        return _LIB
    path = library_path()
    if not os.path.exists(path):
        raise RuntimeError(f"{path} is missing: build it with `python -m qwengine_b200.build` (needs nvcc)")
    lib = C.CDLL(path)
    vp, ll, i32, u32, sz = C.c_void_p, C.c_longlong, C.c_int, C.c_uint32, C.c_size_t
    lib.q38b_ctx_create.argtypes = [i32, C.POINTER(vp)]
    lib.q38b_ctx_destroy.argtypes = [vp]
    lib.q38b_ctx_destroy.restype = None
    lib.q38b_ctx_check.argtypes = [vp, vp]
    lib.q38b_last_cuda_error.argtypes = [vp]
    lib.q38b_ctx_set_pdl.argtypes = [vp, i32]
    lib.q38b_ctx_set_uniform_columns.argtypes = [vp, i32]
    lib.q38b_ctx_set_static_weights.argtypes = [vp, i32]
    lib.q38b_status_string.argtypes = [i32]
    lib.q38b_status_string.restype = C.c_char_p
    lib.q38b_format_supported.argtypes = [u32]
    lib.q38b_row_bytes.argtypes = [u32, i32]
    lib.q38b_row_bytes.restype = sz
    lib.q38b_q8k_bytes.argtypes = [i32]
    lib.q38b_q8k_bytes.restype = sz
    lib.q38b_quantize_q8k.argtypes = [vp, vp, ll, i32, i32, vp, ll, vp]
    lib.q38b_gemv_q8k.argtypes = [vp, u32, vp, sz, i32, i32, vp, ll, i32, vp, ll, i32, vp]
    lib.q38b_swiglu_q8k.argtypes = [vp, vp, vp, ll, i32, i32, vp, vp, ll, vp]
    lib.q38b_dequant_rows.argtypes = [vp, u32, vp, sz, i32, i32, vp, i32, vp]
    lib.q38b_gemv_f32.argtypes = [vp, u32, vp, sz, i32, i32, vp, ll, i32, vp, ll, i32, vp, sz, vp]
    lib.q38b_gemv_f32_static.argtypes = [vp, u32, vp, sz, i32, i32, vp, ll, i32, vp, ll, i32, vp]
    lib.q38b_gemv_f32_static_capacity.restype = sz
    lib.q38b_gemm_prefill.argtypes = [vp, u32, vp, sz, i32, i32, vp, ll, i32, vp, ll, i32, vp]
    lib.q38b_gemm_prefill_f16.argtypes = [vp, u32, vp, sz, i32, i32, vp, ll, i32, vp, ll, i32, vp]
    lib.q38b_comm_unique_id.argtypes = [vp]
    lib.q38b_comm_init.argtypes = [vp, i32, i32, vp]
    lib.q38b_peer_arena_create.argtypes = [vp, sz, vp]
    lib.q38b_peer_connect.argtypes = [vp, i32, i32, vp]
    lib.q38b_peer_barrier.argtypes = [vp, vp]
    lib.q38b_pass_op_barrier.argtypes = [vp]
    lib.q38b_pass_set_peer_store.argtypes = [vp, i32]
    lib.q38b_pass_create.argtypes = [vp, i32, C.POINTER(vp)]
    lib.q38b_pass_destroy.argtypes = [vp]
    lib.q38b_pass_destroy.restype = None
    lib.q38b_pass_buffer_f32.argtypes = [vp, i32]
    lib.q38b_pass_buffer_q8k.argtypes = [vp, i32]
    lib.q38b_pass_buffer_ptr.argtypes = [vp, i32]
    lib.q38b_pass_buffer_ptr.restype = vp
    lib.q38b_pass_matrix_upload.argtypes = [vp, u32, vp, sz, i32, i32, i32, i32]
    lib.q38b_pass_matrix_device.argtypes = [vp, u32, vp, sz, i32, i32]
    lib.q38b_pass_op_quantize.argtypes = [vp, i32, i32, i32, i32]
    lib.q38b_pass_op_gemv.argtypes = [vp, i32, i32, i32, i32]
    lib.q38b_pass_op_gemv_local.argtypes = [vp, i32, i32, i32, i32]
    lib.q38b_pass_op_swiglu.argtypes = [vp, i32, i32, i32, i32, i32, i32]
    lib.q38b_pass_op_allgather.argtypes = [vp, i32, i32, i32]
    lib.q38b_pass_run.argtypes = [vp, i32, vp]
    lib.q38b_pass_run_host.argtypes = [vp, i32, i32, vp, i32, i32, i32, vp, i32, vp]
    lib.q38b_pass_weight_bytes.argtypes = [vp]
    lib.q38b_pass_weight_bytes.restype = ll
    lib.q38b_pass_kernel_count.argtypes = [vp]
    lib.q38b_pass_set_merge.argtypes = [vp, i32]
    lib.q38b_add_rmsnorm_q8k.argtypes = [vp, vp, vp, vp, vp, i32, ll, i32, C.c_float, vp, vp, ll, vp]
    lib.q38b_gemv_bf16.argtypes = [vp, vp, i32, i32, vp, vp, vp]
    lib.q38b_swiglu_rows_inplace.argtypes = [vp, vp, vp, i32, i32, ll, i32, vp]
    lib.q38b_topk.argtypes = [vp, vp, ll, i32, i32, i32, i32, vp, vp, i32, vp]
    lib.q38b_pass_op_topk.argtypes = [vp, i32, i32, i32, i32, i32]
    lib.q38b_gguf_open.argtypes = [C.c_char_p, C.POINTER(vp)]
    lib.q38b_gguf_close.argtypes = [vp]
    lib.q38b_gguf_find.argtypes = [vp, C.c_char_p]
    lib.q38b_pass_matrix_from_gguf.argtypes = [vp, vp, i32, i32, i32]
    lib.q38b_ctx_set_wait_budget_cycles.argtypes = [vp, ll]
    lib.q38b_debug_fake_silent_peer.argtypes = [vp, i32]
    lib.q38b_quantize_act_q8.argtypes = [vp, vp, i32, i32, vp, vp, vp, vp]
    lib.q38b_gemv_act_q8.argtypes = [vp, u32, vp, sz, i32, i32, vp, vp, i32, i32, vp, i32, i32, vp]
    lib.q38b_debug_set_rowgroup.argtypes = [vp, i32]
    lib.q38b_debug_occupancy_shortfalls.argtypes = [vp, i32]
    lib.q38b_debug_set_one_cta.argtypes = [vp, i32]
    lib.q38b_debug_set_gemv_part_items.argtypes = [vp, ll]
    lib.q38b_gemv_group.argtypes = [vp, u32, i32, vp, sz, i32, vp, vp, vp, vp, vp]
    lib.q38b_qk_norm_rope.argtypes = [vp, vp, vp, i32, i32, i32, C.c_float, C.c_float, vp, vp, i32, i32, i32, vp]
    lib.q38b_adjust_logits.argtypes = [vp, vp, ll, i32, i32, i32, vp, vp, ll, vp]
    lib.q38b_pass_op_qk_norm_rope.argtypes = [vp, vp, vp, i32, i32, i32, C.c_float, C.c_float, vp, vp]
    lib.q38b_pass_op_adjust_logits.argtypes = [vp, i32, i32, i32, vp, i32, i32]
    lib.q38b_pass_op_adjust_logits_at.argtypes = [vp, i32, i32, i32, i32, vp, i32, i32]
    lib.q38b_mx4_scale_bytes.argtypes = [i32, i32]
    lib.q38b_mx4_scale_bytes.restype = sz
    lib.q38b_quantize_mx4.argtypes = [vp, vp, i32, ll, i32, i32, vp, ll, vp, vp]
    lib.q38b_mx4_tile_scales.argtypes = [vp, vp, ll, i32, i32, vp, vp]
    lib.q38b_dequant_mx4.argtypes = [vp, vp, ll, vp, i32, i32, vp, i32, ll, vp]
    lib.q38b_gemm_mx4.argtypes = [vp, vp, ll, vp, i32, i32, vp, ll, vp, i32, vp, i32, ll, i32, vp]
    lib.q38b_gemm_mx4_scratch_bytes.argtypes = [i32, i32]
    lib.q38b_gemm_mx4_scratch_bytes.restype = sz
    lib.q38b_debug_set_mx4_pairs.argtypes = [vp, i32]
    lib.q38b_debug_set_mx4_two_launches.argtypes = [vp, i32]
    lib.q38b_gemm_mx4_x.argtypes = [vp, vp, ll, vp, i32, i32, vp, i32, ll, i32, vp, i32, ll, i32, vp, sz, vp]
    _LIB = lib
    return lib


def status_string(status):
    return load_library().q38b_status_string(int(status)).decode()


def _stream():
    """The current stream's handle.  Asked for raw: torch.cuda.current_stream() builds a Stream object on every call."""
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


# q38b_heads and q38b_logit_rules as bytes: a call costs a host microsecond less than with ctypes structures
_pack_heads = struct.Struct("@PPqqqqPi4x").pack      # src, dst, src_row, src_head, dst_row, dst_head, weight, n_heads
_pack_rules = struct.Struct("@PPPPPPPPqP").pack      # penalties .. bias_begin, masks, mask_ld, mask_of_row
_pack_pass_heads = struct.Struct("@7i4xP").pack      # q38b_pass_heads: src, src_off, src_head, dst, dst_off, dst_head, n_heads, weight
_empty = torch.empty_strided
_F32, _F64, _I32, _I64, _U8 = torch.float32, torch.float64, torch.int32, torch.int64, torch.uint8
_current_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _need(ok, what):
    if not ok:
        raise ValueError(what)


class Mx4:
    """A matrix in microscaled 4-bit floating point: codes uint8 [rows, K / 2] (two elements a byte), scales uint8 in the library's tiles
    (Context.quantize_mx4 makes both, Context.pack_mx4 takes another producer's)."""
    __slots__ = ("codes", "scales", "rows", "K", "ld")

    def __init__(self, codes, scales):
        rows, half = codes.shape
        ld, one = codes.stride()
        if codes.dtype != _U8 or scales.dtype != _U8 or one != 1:
            raise ValueError("Mx4: uint8 codes [rows, K / 2] with packed rows, uint8 scales")
        if rows < 1 or half < 16 or half % 16:
            raise ValueError("Mx4: K a multiple of 32, at least one row")
        if not scales.is_contiguous() or scales.numel() != ((rows + 127) // 128) * ((half + 63) // 64) * 512:
            raise ValueError("Mx4: contiguous tiles of 128 rows x 4 blocks of scales")
        if codes.get_device() != scales.get_device():
            raise ValueError("Mx4: codes and scales on one device")
        self.codes, self.scales, self.rows, self.K = codes, scales, rows, 2 * half
        self.ld = ld if rows > 1 else half   # (the stride of a single row says nothing)


class Context:
    """One per process and GPU (q38b_ctx)."""

    def __init__(self, device=0):
        self.lib = load_library()
        if not torch.cuda.is_available():
            raise RuntimeError("no CUDA device: this library has no CPU path")
        self.device, self._index = torch.device("cuda", device), device
        h = C.c_void_p()
        rc = self.lib.q38b_ctx_create(device, C.byref(h))
        if rc:
            raise Q38BError(rc, "q38b_ctx_create")
        self.h = h

    def close(self):
        if getattr(self, "h", None):
            self.lib.q38b_ctx_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _rc(self, rc, what):
        if rc:
            if rc == -4:
                what += f" [cudaError {self.lib.q38b_last_cuda_error(self.h)}]"
            raise Q38BError(rc, what)

    def check(self):
        """Synchronises the current stream and raises if a kernel reported a bounded wait that ran out."""
        self._rc(self.lib.q38b_ctx_check(self.h, _stream()), "q38b_ctx_check")

    def peer_arena_create(self, nbytes=256 << 20):
        """Allocates this rank's peer-visible arena; returns its 64-byte CUDA IPC handle."""
        raw = (C.c_ubyte * 64)()
        self._rc(self.lib.q38b_peer_arena_create(self.h, nbytes, raw), "q38b_peer_arena_create")
        return bytes(raw)

    def peer_connect(self, n_ranks, rank, handles):
        self._rc(self.lib.q38b_peer_connect(self.h, n_ranks, rank, b"".join(handles)), "q38b_peer_connect")

    def set_static_weights(self, enabled):
        self._rc(self.lib.q38b_ctx_set_static_weights(self.h, int(bool(enabled))), "q38b_ctx_set_static_weights")

    def set_uniform_columns(self, enabled):
        self._rc(self.lib.q38b_ctx_set_uniform_columns(self.h, int(bool(enabled))), "q38b_ctx_set_uniform_columns")

    def debug_set_rowgroup(self, enabled):
        """Test hook: enabled=False keeps the one-column kernel on its lane-per-granule mapping for every format."""
        self._rc(self.lib.q38b_debug_set_rowgroup(self.h, int(bool(enabled))), "q38b_debug_set_rowgroup")

    def debug_set_one_cta(self, mode):
        """Test hook: one CTA per SM for the one-column kernel: 0 never, otherwise wherever such a plan fits (default)."""
        self._rc(self.lib.q38b_debug_set_one_cta(self.h, int(mode)), "q38b_debug_set_one_cta")

    def debug_set_gemv_part_items(self, items):
        """Test hook: the multi-column kernel's K-part scratch area counts as `items` (tile, part) sums (0: its real size)."""
        self._rc(self.lib.q38b_debug_set_gemv_part_items(self.h, int(items)), "q38b_debug_set_gemv_part_items")

    def debug_set_mx4_pairs(self, mode):
        """Test hook: 4-bit products in pairs of CTAs never (-1), with tiles of `mode` tokens, by the rule (0)."""
        self._rc(self.lib.q38b_debug_set_mx4_pairs(self.h, int(mode)), "q38b_debug_set_mx4_pairs")

    def set_wait_budget_cycles(self, cycles):
        self._rc(self.lib.q38b_ctx_set_wait_budget_cycles(self.h, int(cycles)), "q38b_ctx_set_wait_budget_cycles")

    def set_pdl(self, enabled):
        self._rc(self.lib.q38b_ctx_set_pdl(self.h, int(bool(enabled))), "q38b_ctx_set_pdl")

    # ---- activations -------------------------------------------------------------------------
    def quantize_q8k(self, x, out=None):
        """x float32 [nb, K] (row stride = x.stride(0)) -> uint8 [nb, K/256*292] of Q8_K blocks."""
        assert x.is_cuda and x.dtype == torch.float32 and x.dim() == 2 and x.stride(1) == 1
        nb, K = x.shape
        if out is None:
            out = torch.empty((nb, K // 256 * F.Q8K_BLOCK_BYTES), dtype=torch.uint8, device=x.device)
        self._rc(self.lib.q38b_quantize_q8k(self.h, x.data_ptr(), x.stride(0), K, nb, out.data_ptr(),
                                            out.stride(0) // F.Q8K_BLOCK_BYTES, _stream()), "q38b_quantize_q8k")
        return out

    def swiglu_q8k(self, g, u, want_h=True, want_q=True):
        """h = silu(g) * u for float32 [nb, n]; returns (h or None, q8k blocks or None)."""
        assert g.shape == u.shape and g.stride() == u.stride() and g.stride(1) == 1
        nb, n = g.shape
        h = torch.empty_like(g) if want_h else None
        q = torch.empty((nb, n // 256 * F.Q8K_BLOCK_BYTES), dtype=torch.uint8, device=g.device) if want_q else None
        if h is not None:
            assert h.stride() == g.stride()
        self._rc(self.lib.q38b_swiglu_q8k(self.h, g.data_ptr(), u.data_ptr(), g.stride(0), n, nb,
                                          h.data_ptr() if h is not None else None,
                                          q.data_ptr() if q is not None else None,
                                          (q.stride(0) // F.Q8K_BLOCK_BYTES) if q is not None else 0, _stream()),
                 "q38b_swiglu_q8k")
        return h, q

    # ---- matvec ------------------------------------------------------------------------------
    def gemv(self, fmt, W, xq, K, out=None, accumulate=False, M=None):
        """W uint8 [M, row_bytes]; xq uint8 [nb, K/256*292]; returns y float32 [nb, M] (y[c, r])."""
        _need(out is not None or not accumulate, "gemv: accumulate needs an out to add to")
        f = F.get(fmt)
        assert W.is_cuda and W.dtype == torch.uint8 and W.dim() == 2 and W.stride(1) == 1
        M = W.shape[0] if M is None else M
        nb = xq.shape[0]
        if out is None:
            out = torch.empty((nb, M), dtype=torch.float32, device=W.device)
        self._rc(self.lib.q38b_gemv_q8k(self.h, f.type_id, W.data_ptr(), W.stride(0), K, M, xq.data_ptr(),
                                        xq.stride(0) // F.Q8K_BLOCK_BYTES, nb, out.data_ptr(), out.stride(0),
                                        int(bool(accumulate)), _stream()), "q38b_gemv_q8k")
        return out

    def quantize_act_q8(self, x):
        """x float32 [n_rows, K] -> (q int8 [n_rows, K], d float32 [n_rows, K/32], s float32 [n_rows, K/32]): the per-32
        activation format of the reference GPU path."""
        assert x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()
        n, K = x.shape
        q = torch.empty((n, K), dtype=torch.int8, device=x.device)
        d = torch.empty((n, K // 32), dtype=torch.float32, device=x.device)
        s = torch.empty_like(d)
        self._rc(self.lib.q38b_quantize_act_q8(self.h, x.data_ptr(), K, n, q.data_ptr(), d.data_ptr(), s.data_ptr(), _stream()),
                 "q38b_quantize_act_q8")
        return q, d, s

    def gemv_act_q8(self, fmt, W, q, d, K, out=None, accumulate=False):
        """W uint8 [M, row_bytes]; q int8 [nb, K], d float32 [nb, K/32] (contiguous); returns y float32 [nb, M]."""
        _need(out is not None or not accumulate, "gemv_act_q8: accumulate needs an out to add to")
        f = F.get(fmt)
        M, nb = W.shape[0], q.shape[0]
        if out is None:
            out = torch.empty((nb, M), dtype=torch.float32, device=W.device)
        self._rc(self.lib.q38b_gemv_act_q8(self.h, f.type_id, W.data_ptr(), W.stride(0), K, M, q.data_ptr(), d.data_ptr(), nb,
                                           q.stride(0), out.data_ptr(), out.stride(0), int(bool(accumulate)), _stream()),
                 "q38b_gemv_act_q8")
        return out

    def add_rmsnorm_q8k(self, x, w, a=None, b=None, eps=1e-6, want_xn=True):
        """x float32 [rows, n] (updated in place when a or b is given); returns (xn float32 or None, q8k uint8 [rows, n/256*292])."""
        rows, n = x.shape
        xn = torch.empty_like(x) if want_xn else None
        q8 = torch.empty((rows, n // 256 * F.Q8K_BLOCK_BYTES), dtype=torch.uint8, device=x.device)
        ptr = lambda t: t.data_ptr() if t is not None else None
        self._rc(self.lib.q38b_add_rmsnorm_q8k(self.h, x.data_ptr(), ptr(a), ptr(b), w.data_ptr(), n, x.stride(0), rows, eps, ptr(xn),
                                               q8.data_ptr(), n // 256, _stream()), "q38b_add_rmsnorm_q8k")
        return xn, q8

    def gemv_bf16(self, W, x):
        """W bfloat16 [N, K], x float32 [K] -> y float32 [N]."""
        N, K = W.shape
        y = torch.empty(N, dtype=torch.float32, device=W.device)
        self._rc(self.lib.q38b_gemv_bf16(self.h, W.data_ptr(), K, N, x.data_ptr(), y.data_ptr(), _stream()), "q38b_gemv_bf16")
        return y

    # ---- the steps of a token between its products --------------------------------------------
    def _stream(self):
        """The current stream of the context's device (whatever device is current)."""
        return _current_stream(self._index)

    def qk_norm_rope(self, q, k, positions, inv_freq, q_weight=None, k_weight=None, eps=1e-6, adjacent=False, scale=1.0, kind=None, q_out=None, k_out=None):
        """q [rows, heads, D], k [rows, heads, D] or None (fp32, fp16 or bf16, any row and head strides): RMSNorm of each head, rotation of its first
        2 * len(inv_freq) elements by positions (int32 [rows]) times inv_freq (float64); weights fp32 [D].  kind: OUT_* of the results (that of
        the inputs by default); returns (q_out, k_out), which may be q and k themselves."""
        rows, _, D = q.shape
        dtype, dev = q.dtype, self._index
        in_kind = _OUT_KINDS.get(dtype)
        if in_kind is None:
            raise ValueError("qk_norm_rope: fp32, fp16 or bf16 heads")
        if kind is None:
            kind = in_kind
        out_dtype, rot, pos_ptr, freq_ptr = _OUT_DTYPES[kind], 0, None, None
        if inv_freq is not None and inv_freq.numel():
            rot = 2 * inv_freq.numel()
            if positions is None or positions.dtype != _I32 or positions.numel() != rows or not positions.is_contiguous():
                raise ValueError("qk_norm_rope: int32 positions, one per row")
            if inv_freq.dtype != _F64 or not inv_freq.is_contiguous() or rot > D:
                raise ValueError("qk_norm_rope: float64 inv_freq, at most D / 2")
            if positions.get_device() != dev or inv_freq.get_device() != dev:
                raise ValueError("qk_norm_rope: tensors on the context's device")
            pos_ptr, freq_ptr = positions.data_ptr(), inv_freq.data_ptr()
        q_out, q_part = self._heads(q, q_weight, q_out, rows, D, dtype, out_dtype, dev)
        k_part = None
        if k is not None:
            k_out, k_part = self._heads(k, k_weight, k_out, rows, D, dtype, out_dtype, dev)
        rc = self.lib.q38b_qk_norm_rope(self.h, q_part, k_part, D, rot, 1 if adjacent else 0, eps, scale, pos_ptr, freq_ptr, in_kind, kind, rows, _current_stream(dev))
        if rc:
            self._rc(rc, "q38b_qk_norm_rope")
        return q_out, k_out if k is not None else None

    def _heads(self, x, w, out, rows, D, dtype, out_dtype, dev):
        """Checks one tensor of heads: its output, and the bytes of its q38b_heads."""
        n, heads, d = x.shape
        row, head, one = x.stride()
        if n != rows or d != D or x.dtype != dtype or (one != 1 and D != 1):
            raise ValueError("qk_norm_rope: heads [rows, heads, D] of one type, elements side by side")
        if out is None:
            out_row, out_head = heads * D, D
            out = _empty((rows, heads, D), (out_row, D, 1), dtype=out_dtype, device=self.device)
        else:
            out_row, out_head, one = out.stride()
            if out.shape != x.shape or out.dtype != out_dtype or (one != 1 and D != 1):
                raise ValueError("qk_norm_rope: outputs shaped like the heads")
        if x.get_device() != dev or out.get_device() != dev:
            raise ValueError("qk_norm_rope: tensors on the context's device")
        w_ptr = 0
        if w is not None:
            if w.dtype != _F32 or w.numel() != D or not w.is_contiguous() or w.get_device() != dev:
                raise ValueError("qk_norm_rope: fp32 weights [D] on the context's device")
            w_ptr = w.data_ptr()
        return out, _pack_heads(x.data_ptr(), out.data_ptr(), row, head, out_row, out_head, w_ptr, heads)

    def _list(self, what, t, dtype, shape=None):
        """Address of an optional contiguous tensor of the context's device (0: none, or nothing in it)."""
        if t is None:
            return 0
        if t.dtype != dtype or not t.is_contiguous() or t.get_device() != self._index or (shape is not None and t.shape != shape):
            raise ValueError(what)
        return t.data_ptr()

    def logit_rules(self, rows, n, penalties=None, history=None, history_begin=None, prompt_len=None, bias_ids=None, bias_values=None, bias_begin=None,
                    masks=None, mask_of_row=None, index_offset=0):
        """The bytes of a q38b_logit_rules of checked device tensors: penalties fp32 [rows, 3] (repetition, frequency, presence), history int32 with int64
        begins [rows + 1] and int32 prompt lengths [rows]; bias_ids int32, bias_values fp32, int64 begins; masks int32 [*, words] of
        allowed-token bits, mask_of_row int32 [rows]."""
        f32, i32, i64, address = _F32, _I32, _I64, self._list
        p = h = hb = pl = bi = bv = bb = mk = mr = ld = 0
        if penalties is not None or history is not None or history_begin is not None or prompt_len is not None:
            p = address("adjust_logits: fp32 penalties [rows, 3]", penalties, f32, (rows, 3))
            h = address("adjust_logits: int32 history", history, i32)
            hb = address("adjust_logits: int64 history_begin [rows + 1]", history_begin, i64, (rows + 1,))
            pl = address("adjust_logits: int32 prompt_len [rows]", prompt_len, i32, (rows,))
            if history is not None and history.numel() == 0:
                p = h = hb = pl = 0   # no token at all: nothing to penalise
        if bias_ids is not None or bias_values is not None or bias_begin is not None:
            bi = address("adjust_logits: int32 bias_ids", bias_ids, i32)
            bv = address("adjust_logits: fp32 bias_values", bias_values, f32)
            bb = address("adjust_logits: int64 bias_begin [rows + 1]", bias_begin, i64, (rows + 1,))
            if bias_ids is not None:
                _need(bias_values is not None and bias_values.numel() == bias_ids.numel(), "adjust_logits: one value per bias")
                if bias_ids.numel() == 0:
                    bi = bv = bb = 0
        if masks is not None:
            count, words = masks.shape
            ld, one = masks.stride()
            _need(masks.dtype == i32 and one == 1 and masks.get_device() == self._index and words * 32 >= index_offset + n and
                  (count >= rows or mask_of_row is not None), "adjust_logits: masks int32 [masks, words], a bit for each token")
            mk, ld = masks.data_ptr(), ld if count > 1 else words
        if mask_of_row is not None:
            mr = address("adjust_logits: mask_of_row int32 [rows]", mask_of_row, i32, (rows,))
        return _pack_rules(p, h, hb, pl, bi, bv, bb, mk, ld, mr)

    def adjust_logits(self, logits, out=None, index_offset=0, **rules):
        """logits fp32 [rows, n] (rows any distance of n and more apart) -> penalised, biased, masked logits (`out`, which may be `logits`); the rules are those of
        logit_rules.  Token v is column v - index_offset."""
        rows, n = logits.shape
        ld, one = logits.stride()
        dev = self._index
        if logits.dtype != _F32 or (one != 1 and n != 1) or logits.get_device() != dev:
            raise ValueError("adjust_logits: fp32 logits [rows, n] on the context's device")
        r = self.logit_rules(rows, n, index_offset=index_offset, **rules)
        if out is None:
            out_ld = n
            out = _empty((rows, n), (n, 1), dtype=torch.float32, device=self.device)
        else:
            out_ld, one = out.stride()
            _need(out.dtype == torch.float32 and out.shape == logits.shape and (one == 1 or n == 1) and out.get_device() == dev, "adjust_logits: fp32 out of the logits' shape")
        rc = self.lib.q38b_adjust_logits(self.h, logits.data_ptr(), ld, n, rows, index_offset, r, out.data_ptr(), out_ld, _current_stream(dev))
        if rc:
            self._rc(rc, "q38b_adjust_logits")
        return out

    # ---- microscaled 4-bit floating point -----------------------------------------------------
    def quantize_mx4(self, x):
        """x [rows, K] (fp32, fp16 or bf16, rows any distance of K and more apart) -> Mx4."""
        rows, K = x.shape
        ld, one = x.stride()
        kind = _OUT_KINDS.get(x.dtype)
        if kind is None or one != 1 or x.get_device() != self._index:
            raise ValueError("quantize_mx4: fp32, fp16 or bf16 [rows, K] on the context's device")
        if K % 32 or K == 0 or rows == 0:
            raise Q38BError(-1, "q38b_quantize_mx4")
        half, tiles = K // 2, ((rows + 127) // 128) * ((K + 127) // 128) * 512
        codes = _empty((rows, half), (half, 1), dtype=torch.uint8, device=self.device)
        scales = _empty((tiles,), (1,), dtype=torch.uint8, device=self.device)
        rc = self.lib.q38b_quantize_mx4(self.h, x.data_ptr(), kind, ld if rows > 1 else K, K, rows, codes.data_ptr(), half, scales.data_ptr(), _current_stream(self._index))
        if rc:
            self._rc(rc, "q38b_quantize_mx4")
        m = Mx4.__new__(Mx4)   # (made here: nothing to check)
        m.codes, m.scales, m.rows, m.K, m.ld = codes, scales, rows, K, half
        return m

    def pack_mx4(self, codes, scales):
        """Codes uint8 [rows, K / 2] and scale bytes uint8 [rows, K / 32] of another producer -> Mx4 (the codes are kept, not copied)."""
        rows, half = codes.shape
        _need(scales.dtype == torch.uint8 and scales.shape == (rows, half // 16) and half % 16 == 0 and scales.stride(1) == 1, "pack_mx4: uint8 scales [rows, K / 32]")
        _need(codes.get_device() == self._index and scales.get_device() == self._index, "pack_mx4: tensors on the context's device")
        K = 2 * half
        tiles = torch.empty(self.lib.q38b_mx4_scale_bytes(K, rows), dtype=torch.uint8, device=self.device)
        self._rc(self.lib.q38b_mx4_tile_scales(self.h, scales.data_ptr(), scales.stride(0) if rows > 1 else K // 32, K, rows, tiles.data_ptr(), self._stream()), "q38b_mx4_tile_scales")
        return Mx4(codes, tiles)

    def dequant_mx4(self, m, kind=OUT_F32):
        """The values of an Mx4: [rows, K]."""
        codes, rows, K = m.codes, m.rows, m.K
        if codes.get_device() != self._index:
            raise ValueError("dequant_mx4: a matrix on the context's device")
        out = _empty((rows, K), (K, 1), dtype=_OUT_DTYPES[kind], device=self.device)
        rc = self.lib.q38b_dequant_mx4(self.h, codes.data_ptr(), m.ld, m.scales.data_ptr(), K, rows, out.data_ptr(), kind, K, _current_stream(self._index))
        if rc:
            self._rc(rc, "q38b_dequant_mx4")
        return out

    def gemm_mx4(self, W, X, kind=OUT_F32, out=None, accumulate=False):
        """Y [B, W.rows] = X W^T for W an Mx4 and X an Mx4 or activations [B, K] (fp32, fp16 or bf16), which are quantized first.  kind: OUT_* of Y
        where `out` is not given; accumulate adds to `out`."""
        _need(out is not None or not accumulate, "gemm_mx4: accumulate needs an out to add to")
        K, M, dev, mx = W.K, W.rows, self._index, isinstance(X, Mx4)
        B = X.rows if mx else X.shape[0]
        if W.codes.get_device() != dev or (X.codes if mx else X).get_device() != dev:
            raise ValueError("gemm_mx4: operands on the context's device")
        if out is None:
            ldy = M
            out = _empty((B, M), (M, 1), dtype=_OUT_DTYPES[kind], device=self.device)
        else:
            kind = _OUT_KINDS.get(out.dtype)
            _need(kind is not None and out.shape == (B, M) and (M == 1 or out.stride(1) == 1) and out.get_device() == dev, "gemm_mx4: out [B, W.rows]")
            ldy = out.stride(0) if B > 1 else M
        if mx:
            _need(X.K == K, "gemm_mx4: operands of one K")
            rc = self.lib.q38b_gemm_mx4(self.h, W.codes.data_ptr(), W.ld, W.scales.data_ptr(), K, M, X.codes.data_ptr(), X.ld, X.scales.data_ptr(), B, out.data_ptr(), kind,
                                        ldy, 1 if accumulate else 0, self._stream())
            if rc:
                self._rc(rc, "q38b_gemm_mx4")
            return out
        x_kind = _OUT_KINDS.get(X.dtype)
        B, k = X.shape
        ld, one = X.stride()
        if x_kind is None or one != 1 or k != K or B == 0:
            raise ValueError("gemm_mx4: activations [B, K] of the weights' K")
        scratch, need = None, 0
        if B > 1 or K > 8192:   # q38b_gemm_mx4_scratch_bytes
            need = B * (K // 2) + ((B + 127) // 128) * ((K + 127) // 128) * 512 + 16
            scratch = _empty((need,), (1,), dtype=torch.uint8, device=self.device)
        rc = self.lib.q38b_gemm_mx4_x(self.h, W.codes.data_ptr(), W.ld, W.scales.data_ptr(), K, M, X.data_ptr(), x_kind, ld if B > 1 else K, B, out.data_ptr(), kind, ldy,
                                      1 if accumulate else 0, None if scratch is None else scratch.data_ptr(), need, self._stream())
        if rc:
            self._rc(rc, "q38b_gemm_mx4_x")
        return out

    def topk(self, logits, k, index_offset=0):
        """The k largest of each row of `logits` [rows, n] (fp32, device): (values [rows, k], positions [rows, k] int32)."""
        rows, n = logits.shape
        vals = torch.empty((rows, k), dtype=torch.float32, device=logits.device)
        idx = torch.empty((rows, k), dtype=torch.int32, device=logits.device)
        self._rc(self.lib.q38b_topk(self.h, logits.data_ptr(), logits.stride(0), n, rows, k, index_offset, vals.data_ptr(),
                                    idx.data_ptr(), k, _stream()), "q38b_topk")
        return vals, idx

    def swiglu_rows_inplace(self, G, U, n, kind):
        """G, U float32 [B, ld]; writes silu(G[:, :n]) * U[:, :n] over the start of every row of G as 16-bit floats."""
        self._rc(self.lib.q38b_swiglu_rows_inplace(self.h, G.data_ptr(), U.data_ptr(), G.shape[0], n, G.stride(0), kind, _stream()),
                 "q38b_swiglu_rows_inplace")

    def gemv_group(self, fmt, Ws, K, xq=None, x_f32=None):
        """q38b_gemv_group: up to three matrices [M_i, row_bytes] of one format on one column, given as Q8_K blocks
        (xq uint8 [1, K/256*292]) or as floats (x_f32 [K] or [1, K]); returns the list of y_i float32 [M_i]."""
        import ctypes
        f = F.get(fmt)
        n = len(Ws)
        outs = [torch.empty(w.shape[0], dtype=torch.float32, device=w.device) for w in Ws]
        Wp = (ctypes.c_void_p * n)(*[w.data_ptr() for w in Ws])
        yp = (ctypes.c_void_p * n)(*[o.data_ptr() for o in outs])
        Ms = (ctypes.c_int * n)(*[w.shape[0] for w in Ws])
        self._rc(self.lib.q38b_gemv_group(self.h, f.type_id, n, Wp, Ws[0].stride(0), K, Ms, xq.data_ptr() if xq is not None else None,
                                          x_f32.data_ptr() if x_f32 is not None else None, yp, _stream()), "q38b_gemv_group")
        return outs

    def gemv_f32(self, fmt, W, x, K, scratch=None, out=None, accumulate=False):
        """Matvec from fp32 activations x [nb, K]; `scratch` is a uint8 device tensor for the Q8_K blocks."""
        _need(out is not None or not accumulate, "gemv_f32: accumulate needs an out to add to")
        f = F.get(fmt)
        nb, M = x.shape[0], W.shape[0]
        if scratch is None:
            scratch = torch.empty(nb * (K // 256) * F.Q8K_BLOCK_BYTES, dtype=torch.uint8, device=W.device)
        if out is None:
            out = torch.empty((nb, M), dtype=torch.float32, device=W.device)
        self._rc(self.lib.q38b_gemv_f32(self.h, f.type_id, W.data_ptr(), W.stride(0), K, M, x.data_ptr(), x.stride(0), nb,
                                        out.data_ptr(), out.stride(0), int(bool(accumulate)), scratch.data_ptr(), scratch.numel(),
                                        _stream()), "q38b_gemv_f32")
        return out

    def gemv_f32_static(self, fmt, W, x, K, out=None, accumulate=False):
        """q38b_gemv_f32_static: like gemv_f32 but the Q8_K scratch is the library's built-in array (no allocation)."""
        f = F.get(fmt)
        nb, M = x.shape[0], W.shape[0]
        assert out is not None, "the caller brings the output buffer: this path allocates nothing"
        self._rc(self.lib.q38b_gemv_f32_static(self.h, f.type_id, W.data_ptr(), W.stride(0), K, M, x.data_ptr(), x.stride(0), nb,
                                               out.data_ptr(), out.stride(0), int(bool(accumulate)), _stream()),
                 "q38b_gemv_f32_static")
        return out

    def gemv_raw(self, type_id, W_ptr, row_bytes, K, M, xq_ptr, x_stride, nb, y_ptr, y_ld, accumulate=0):
        """Unchecked pass-through to q38b_gemv_q8k; returns the status code."""
        return self.lib.q38b_gemv_q8k(self.h, type_id, W_ptr, row_bytes, K, M, xq_ptr, x_stride, nb, y_ptr, y_ld,
                                      accumulate, _stream())

    def gemm_prefill(self, fmt, W, X, K, out=None, accumulate=False):
        """W uint8 [M, row_bytes]; X bfloat16 or float16 [B, K] (the operand type of the tensor-core product follows X);
        returns Y float32 [B, M] = X @ dequant(W)^T."""
        _need(out is not None or not accumulate, "gemm_prefill: accumulate needs an out to add to")
        f = F.get(fmt)
        assert X.dtype in (torch.bfloat16, torch.float16) and X.stride(1) == 1
        M, B = W.shape[0], X.shape[0]
        if out is None:
            out = torch.empty((B, M), dtype=torch.float32, device=W.device)
        fn = self.lib.q38b_gemm_prefill if X.dtype == torch.bfloat16 else self.lib.q38b_gemm_prefill_f16
        self._rc(fn(self.h, f.type_id, W.data_ptr(), W.stride(0), K, M, X.data_ptr(), X.stride(0), B,
                    out.data_ptr(), out.stride(0), int(bool(accumulate)), _stream()), "q38b_gemm_prefill")
        return out

    def dequant_rows(self, fmt, W, K, kind=OUT_F32):
        f = F.get(fmt)
        rows = W.shape[0]
        out = torch.empty((rows, K), dtype=_OUT_DTYPES[kind], device=W.device)
        self._rc(self.lib.q38b_dequant_rows(self.h, f.type_id, W.data_ptr(), W.stride(0), K, rows, out.data_ptr(), kind,
                                            _stream()), "q38b_dequant_rows")
        return out


class Pass:
    """Recorded decode pass over resident matrices (q38b_pass): the all-HBM planner's run-time object."""

    def __init__(self, ctx, max_nb=1):
        self.ctx, self.lib, self.max_nb = ctx, ctx.lib, max_nb
        h = C.c_void_p()
        ctx._rc(self.lib.q38b_pass_create(ctx.h, max_nb, C.byref(h)), "q38b_pass_create")
        self.h = h
        self._keep = []          # device tensors adopted with matrix_device stay alive with the pass
        self._sizes = {}

    def close(self):
        if getattr(self, "h", None):
            self.lib.q38b_pass_destroy(self.h)
            self.h = None

    def _id(self, rc, what):
        if rc < 0:
            raise Q38BError(rc, what)
        return rc

    def buffer_f32(self, n):
        i = self._id(self.lib.q38b_pass_buffer_f32(self.h, n), "q38b_pass_buffer_f32")
        self._sizes[i] = n
        return i

    def buffer_q8k(self, K):
        return self._id(self.lib.q38b_pass_buffer_q8k(self.h, K), "q38b_pass_buffer_q8k")

    def buffer_tensor(self, buf):
        """A torch view [max_nb, n] of an fp32 buffer of the pass (no copy)."""
        n = self._sizes[buf]
        ptr = self.lib.q38b_pass_buffer_ptr(self.h, buf)
        return _tensor_from_ptr(ptr, (self.max_nb, n), self.ctx.device)

    def matrix_upload(self, fmt, w_host, K, shard=0, n_shards=1):
        """w_host: numpy uint8 [M, row_bytes] in host memory; uploads rows of this shard."""
        f = F.get(fmt)
        M, rb = w_host.shape
        return self._id(self.lib.q38b_pass_matrix_upload(self.h, f.type_id, w_host.ctypes.data, rb, K, M, shard, n_shards),
                        "q38b_pass_matrix_upload")

    def matrix_from_gguf(self, gguf_file, name, shard=0, n_shards=1):
        """Uploads this rank's rows of the named 2-D tensor of an open GGUF file (GgufFile); returns the matrix id."""
        idx = self.lib.q38b_gguf_find(gguf_file.h, name.encode())
        if idx < 0:
            raise KeyError(name)
        return self._id(self.lib.q38b_pass_matrix_from_gguf(self.h, gguf_file.h, idx, shard, n_shards), "q38b_pass_matrix_from_gguf")

    def matrix_device(self, fmt, W, K):
        f = F.get(fmt)
        self._keep.append(W)
        return self._id(self.lib.q38b_pass_matrix_device(self.h, f.type_id, W.data_ptr(), W.stride(0), K, W.shape[0]),
                        "q38b_pass_matrix_device")

    def quantize(self, src, off, K, dst):
        self.ctx._rc(self.lib.q38b_pass_op_quantize(self.h, src, off, K, dst), "q38b_pass_op_quantize")

    def gemv(self, mat, src_q, dst, off=0, local=False):
        """local=True: the output is not pushed to the peers (a matrix every rank holds whole)."""
        fn = self.lib.q38b_pass_op_gemv_local if local else self.lib.q38b_pass_op_gemv
        self.ctx._rc(fn(self.h, mat, src_q, dst, off), "q38b_pass_op_gemv")

    def swiglu(self, g, g_off, u, u_off, n, dst_q):
        self.ctx._rc(self.lib.q38b_pass_op_swiglu(self.h, g, g_off, u, u_off, n, dst_q), "q38b_pass_op_swiglu")

    def set_peer_store(self, enabled):
        self.ctx._rc(self.lib.q38b_pass_set_peer_store(self.h, int(bool(enabled))), "q38b_pass_set_peer_store")

    def set_merge(self, enabled):
        """enabled=False: single-column runs launch one kernel per recorded step (no shared launches, no folded quantize)."""
        self.ctx._rc(self.lib.q38b_pass_set_merge(self.h, int(bool(enabled))), "q38b_pass_set_merge")

    def topk(self, src, off, n, k, dst):
        self.ctx._rc(self.lib.q38b_pass_op_topk(self.h, src, off, n, k, dst), "q38b_pass_op_topk")

    def qk_norm_rope(self, q, k, D, positions, inv_freq, q_weight=None, k_weight=None, eps=1e-6, adjacent=False, scale=1.0):
        """q, k (or None): dicts of buf, n_heads and, if need be, off (0), head (D), dst (buf: in place), dst_off, dst_head.  positions int32
        [max_nb], inv_freq float64 and weights fp32 [D] are device tensors, kept by the pass and read at every run."""
        for t, dtype, shape in ((positions, torch.int32, (self.max_nb,)), (inv_freq, torch.float64, None), (q_weight, torch.float32, (D,)), (k_weight, torch.float32, (D,))):
            _need(t is None or (t.dtype == dtype and t.is_contiguous() and t.device == self.ctx.device and (shape is None or t.shape == shape)), "qk_norm_rope: device tensors of the pass")
        def pack(h, w):
            off, head, dst = h.get("off", 0), h.get("head", D), h.get("dst", h["buf"])
            here = dst == h["buf"]
            return _pack_pass_heads(h["buf"], off, head, dst, h.get("dst_off", off if here else 0), h.get("dst_head", head if here else D), h["n_heads"], 0 if w is None else w.data_ptr())
        rot = 0 if inv_freq is None else 2 * inv_freq.numel()
        _need(rot == 0 or positions is not None, "qk_norm_rope: positions int32 [max_nb]")
        self.ctx._rc(self.lib.q38b_pass_op_qk_norm_rope(self.h, pack(q, q_weight), None if k is None else pack(k, k_weight), D, rot, int(bool(adjacent)), eps, scale,
                                                        positions.data_ptr() if rot else None, inv_freq.data_ptr() if rot else None), "q38b_pass_op_qk_norm_rope")
        self._keep += [positions, inv_freq, q_weight, k_weight]

    def adjust_logits(self, src, off, n, dst=None, dst_off=None, index_offset=0, **rules):
        """The rules of Context.logit_rules on n logits of buffer src (in place where dst is not given), of which the first is token index_offset's; the
        rules' tensors have max_nb rows, are kept by the pass and read at every run."""
        dst = src if dst is None else dst
        dst_off = (off if dst == src else 0) if dst_off is None else dst_off
        packed = self.ctx.logit_rules(self.max_nb, n, index_offset=index_offset, **rules)
        self.ctx._rc(self.lib.q38b_pass_op_adjust_logits_at(self.h, src, off, n, index_offset, packed, dst, dst_off), "q38b_pass_op_adjust_logits_at")
        self._keep += [t for t in rules.values() if isinstance(t, torch.Tensor)]

    def barrier(self):
        self.ctx._rc(self.lib.q38b_pass_op_barrier(self.h), "q38b_pass_op_barrier")

    def allgather(self, buf, off, count):
        self.ctx._rc(self.lib.q38b_pass_op_allgather(self.h, buf, off, count), "q38b_pass_op_allgather")

    def run(self, nb=1):
        self.ctx._rc(self.lib.q38b_pass_run(self.h, nb, _stream()), "q38b_pass_run")

    def run_host(self, nb, in_buf, x_host, out_buf, out_off, y_host):
        """x_host, y_host: C-contiguous numpy float32 [nb, len]; host to device and back inside the call."""
        self.ctx._rc(self.lib.q38b_pass_run_host(self.h, nb, in_buf, x_host.ctypes.data, x_host.shape[1], out_buf, out_off,
                                                 y_host.ctypes.data, y_host.shape[1], _stream()), "q38b_pass_run_host")

    @property
    def weight_bytes(self):
        return int(self.lib.q38b_pass_weight_bytes(self.h))

    @property
    def kernel_count(self):
        return int(self.lib.q38b_pass_kernel_count(self.h))


class GgufFile:
    """A memory-mapped GGUF model file (q38b_gguf_open)."""

    def __init__(self, path):
        import ctypes
        self.lib = load_library()
        self.h = ctypes.c_void_p()
        rc = self.lib.q38b_gguf_open(str(path).encode(), ctypes.byref(self.h))
        if rc != 0:
            raise Q38BError(rc, "q38b_gguf_open")

    def close(self):
        if self.h:
            self.lib.q38b_gguf_close(self.h)
            self.h = None


def _tensor_from_ptr(ptr, shape, device):
    """Wraps device memory owned by the library as a float32 torch tensor (via __cuda_array_interface__)."""
    class _Holder:
        pass
    h = _Holder()
    h.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": "<f4", "data": (int(ptr), False), "version": 2}
    return torch.as_tensor(h, device=device)
