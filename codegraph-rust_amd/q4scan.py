"""ctypes binding of include/cgvec_q4.h: a corpus in 4 bits with group scales and its scores against a few queries."""
import ctypes as C

import numpy as np

from .cgvec import CGV_ERR_DIM_MISMATCH, CGV_ERR_INVALID_ARG, DTYPES, CgvError, _check, _is_torch, lib as _base_lib, raw_stream, refuse_tangent

_decl = False


def lib():
    global _decl
    L = _base_lib()
    if not _decl:
        vp, u32, u64, i32 = C.c_void_p, C.c_uint32, C.c_uint64, C.c_int
        L.cgv_q4_create.argtypes = [u32, u32, i32, i32, C.POINTER(vp)]
        L.cgv_q4_destroy.argtypes = [vp]
        L.cgv_q4_reserve.argtypes = [vp, u64]
        L.cgv_q4_count.argtypes = [vp]
        L.cgv_q4_count.restype = u64
        L.cgv_q4_add_f32.argtypes = [vp, vp, u64]
        L.cgv_q4_add_f32_dev.argtypes = [vp, vp, u64, vp]
        L.cgv_q4_add_codes.argtypes = [vp, vp, vp, u64]
        L.cgv_q4_add_codes_dev.argtypes = [vp, vp, vp, u64, vp]
        L.cgv_q4_get_row_f32.argtypes = [vp, u64, vp]
        L.cgv_q4_scores_f32.argtypes = [vp, vp, u32, u64, vp]
        L.cgv_q4_scores_dev.argtypes = [vp, vp, i32, u32, u64, vp, vp, C.c_size_t, vp]
        L.cgv_q4_scores_workspace.argtypes = [vp, i32, u32]
        L.cgv_q4_scores_workspace.restype = C.c_size_t
        for n in ("cgv_q4_create", "cgv_q4_destroy", "cgv_q4_reserve", "cgv_q4_add_f32", "cgv_q4_add_f32_dev", "cgv_q4_add_codes",
                  "cgv_q4_add_codes_dev", "cgv_q4_get_row_f32", "cgv_q4_scores_f32", "cgv_q4_scores_dev"):
            getattr(L, n).restype = i32
        _decl = True
    return L


class Int4ScanIndex:
    """Rows kept as 4-bit codes with one scale per `group` elements (32, 64 or 128): value = scale * (code - 8).

    `scales`: "fp16" or "bf16". Rows come as f32 and are quantised on the device (`add`) or already quantised (`add_q4`).
    `scores` is the dot product of each query with every row: queries keep their own precision, sums are f32."""

    def __init__(self, dim, group=64, scales="fp16", device=0):
        self._h = C.c_void_p()
        self.dim, self.group, self.scales, self.device = int(dim), int(group), scales, int(device)
        if scales not in ("fp16", "bf16"):
            raise CgvError(CGV_ERR_INVALID_ARG, f"scales must be 'fp16' or 'bf16', not {scales!r}")
        if self.dim < 1 or self.group < 1:
            raise CgvError(CGV_ERR_INVALID_ARG, "dim must be in 1..=8192 and group 32, 64 or 128")
        h = C.c_void_p()
        _check(lib().cgv_q4_create(self.dim, self.group, DTYPES[scales], self.device, C.byref(h)))
        self._h = h

    def close(self):
        if getattr(self, "_h", None) is not None and self._h:
            lib().cgv_q4_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __len__(self):
        return int(lib().cgv_q4_count(self._h))

    @property
    def n_groups(self):
        return -(-self.dim // self.group)

    def reserve(self, n):
        _check(lib().cgv_q4_reserve(self._h, int(n)))

    def _stream(self):
        return raw_stream(self.device)

    def _on_device(self, t, what):
        if t.device.type != "cuda" or t.device.index != self.device:
            raise CgvError(CGV_ERR_INVALID_ARG, f"{what} is on {t.device}, the index on cuda:{self.device}")

    def add(self, rows):
        """Append [n, dim] rows: numpy / CPU tensors, or CUDA tensors on the index' device (read on torch's current stream)."""
        if _is_torch(rows) and rows.is_cuda:
            import torch
            if rows.dim() != 2 or rows.shape[1] != self.dim:
                raise CgvError(CGV_ERR_DIM_MISMATCH, f"expected [n,{self.dim}] rows, got {tuple(rows.shape)}")
            self._on_device(rows, "rows")
            r = rows.detach().to(torch.float32).contiguous()
            _check(lib().cgv_q4_add_f32_dev(self._h, C.c_void_p(r.data_ptr()), r.shape[0], self._stream()))
            return
        if _is_torch(rows):
            rows = rows.detach().float().numpy()
        r = np.ascontiguousarray(rows, dtype=np.float32)
        if r.ndim != 2 or r.shape[1] != self.dim:
            raise CgvError(CGV_ERR_DIM_MISMATCH, f"expected [n,{self.dim}] rows, got {r.shape}")
        _check(lib().cgv_q4_add_f32(self._h, r.ctypes.data_as(C.c_void_p), r.shape[0]))

    def add_q4(self, codes, scales):
        """Append rows that are already quantised: codes uint8 [n, ceil(dim / 2)], low nibble first, 8 stands for zero; scales
        [n, ceil(dim / group)] in the index' scale type (torch float16 / bfloat16, or numpy float16 / the 16 bits as uint16)."""
        nb = (self.dim + 1) // 2
        if tuple(codes.shape[1:]) != (nb,) or tuple(scales.shape) != (codes.shape[0], self.n_groups):
            raise CgvError(CGV_ERR_DIM_MISMATCH, f"expected codes [n,{nb}] and scales [n,{self.n_groups}], got {tuple(codes.shape)} "
                                                 f"and {tuple(scales.shape)}")
        if _is_torch(codes) != _is_torch(scales):
            raise CgvError(CGV_ERR_INVALID_ARG, "codes and scales must both be torch tensors or both numpy arrays")
        if _is_torch(codes):
            import torch
            want = torch.float16 if self.scales == "fp16" else torch.bfloat16
            if codes.dtype != torch.uint8 or scales.dtype != want:
                raise CgvError(CGV_ERR_INVALID_ARG, f"codes must be uint8 and scales {want}, got {codes.dtype} and {scales.dtype}")
            c, s = codes.detach().contiguous(), scales.detach().contiguous()
            if c.is_cuda or s.is_cuda:
                self._on_device(c, "codes")
                self._on_device(s, "scales")
                _check(lib().cgv_q4_add_codes_dev(self._h, C.c_void_p(c.data_ptr()), C.c_void_p(s.data_ptr()), c.shape[0], self._stream()))
                return
            _check(lib().cgv_q4_add_codes(self._h, C.c_void_p(c.data_ptr()), C.c_void_p(s.data_ptr()), c.shape[0]))
            return
        c = np.ascontiguousarray(codes)
        s = np.ascontiguousarray(scales)
        if c.dtype != np.uint8 or not (s.dtype == np.uint16 or (s.dtype == np.float16 and self.scales == "fp16")):
            raise CgvError(CGV_ERR_INVALID_ARG, f"codes must be uint8 and scales 16-bit, got {c.dtype} and {s.dtype}")
        _check(lib().cgv_q4_add_codes(self._h, c.ctypes.data_as(C.c_void_p), s.ctypes.data_as(C.c_void_p), c.shape[0]))

    def get_row(self, i):
        """The stored row as f32 values."""
        if int(i) < 0:
            raise CgvError(CGV_ERR_INVALID_ARG, "row id must be >= 0")
        out = np.empty(self.dim, dtype=np.float32)
        _check(lib().cgv_q4_get_row_f32(self._h, int(i), out.ctypes.data_as(C.c_void_p)))
        return out

    def scores(self, queries):
        """Dot products with every row, f32: [dim] -> [n], [m, dim] -> [m, n]. Host arrays in, numpy out; a CUDA tensor (f32,
        bf16 or fp16) in, a CUDA tensor out, enqueued on torch's current stream. Not differentiable: the result never requires a
        gradient, also where the queries do."""
        if _is_torch(queries):
            refuse_tangent(queries, "queries")
        if _is_torch(queries) and queries.is_cuda:
            import torch
            code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}.get(queries.dtype)
            if code is None:
                raise CgvError(CGV_ERR_INVALID_ARG, f"queries must be float32, bfloat16 or float16, not {queries.dtype}")
            self._on_device(queries, "queries")
            one = queries.dim() == 1
            q = (queries.detach()[None] if one else queries).contiguous()
            if q.dim() != 2 or q.shape[1] != self.dim:
                raise CgvError(CGV_ERR_DIM_MISMATCH, f"query dim {tuple(queries.shape)} != {self.dim}")
            L, m = lib(), q.shape[0]
            if m >= 1 << 32:
                raise CgvError(CGV_ERR_INVALID_ARG, "more than 2^32 - 1 queries")
            n = L.cgv_q4_count(self._h)
            out = torch.empty((m, n), dtype=torch.float32, device=q.device)
            nb = L.cgv_q4_scores_workspace(self._h, code, m)
            ws = torch.empty((nb,), dtype=torch.uint8, device=q.device) if nb else None
            _check(L.cgv_q4_scores_dev(self._h, q.data_ptr(), code, m, n, out.data_ptr(), ws.data_ptr() if nb else None, nb, self._stream()))
            return out[0] if one else out
        if _is_torch(queries):
            queries = queries.detach().float().numpy()
        q = np.ascontiguousarray(queries, dtype=np.float32)
        one = q.ndim == 1
        q = q[None, :] if one else q
        if q.ndim != 2 or q.shape[1] != self.dim:
            raise CgvError(CGV_ERR_DIM_MISMATCH, f"query dim {q.shape} != {self.dim}")
        out = np.empty((q.shape[0], len(self)), dtype=np.float32)
        _check(lib().cgv_q4_scores_f32(self._h, q.ctypes.data_as(C.c_void_p), q.shape[0], out.shape[1], out.ctypes.data_as(C.c_void_p)))
        return out[0] if one else out
