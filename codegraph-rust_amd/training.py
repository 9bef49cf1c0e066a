"""ctypes binding of include/cgvec_train.h with torch's autograd: rows of a table by id, and the losses that train what an index
serves. CUDA tensors only (there is no CPU fallback); every call enqueues on torch's current stream of the tensors' device and can be captured
into a graph. (A backward pass is captured without eager autograd graphs of the same leaves alive, as torch asks for.)"""
import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from .cgvec import CGV_ERR_DIM_MISMATCH, CGV_ERR_INVALID_ARG, CgvError, _check, lib as _base_lib, raw_stream as _stream, refuse_tangent

_decl = False
_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def lib():
    global _decl
    L = _base_lib()
    if not _decl:
        vp, u32, u64, i32, f32, sz = C.c_void_p, C.c_uint32, C.c_uint64, C.c_int, C.c_float, C.c_size_t
        L.cgv_lookup_rows_dev.argtypes = [i32, vp, i32, u64, u32, u64, vp, u64, f32, vp, vp]
        L.cgv_lookup_grad_workspace.argtypes = [u64, u64, u32]
        L.cgv_lookup_grad_workspace.restype = sz
        L.cgv_lookup_grad_dev.argtypes = [i32, vp, i32, vp, u64, u64, u32, f32, vp, vp, sz, vp]
        for n in ("cgv_corpus_loss_workspace", "cgv_corpus_loss_grad_workspace"):
            getattr(L, n).argtypes = [u64, u64, u32, u32, i32]
            getattr(L, n).restype = sz
        L.cgv_corpus_loss_dev.argtypes = [i32, vp, u64, vp, u64, i32, u64, u64, u32, vp, vp, u32, f32, f32, vp, vp, vp, sz, vp]
        L.cgv_corpus_loss_grad_dev.argtypes = [i32, vp, u64, vp, u64, i32, u64, u64, u32, vp, vp, u32, f32, f32, vp, vp, vp, vp, vp, sz, vp]
        for n in ("cgv_lookup_rows_dev", "cgv_lookup_grad_dev", "cgv_corpus_loss_dev", "cgv_corpus_loss_grad_dev"):
            getattr(L, n).restype = i32
        _decl = True
    return L


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _bad(msg, code=CGV_ERR_INVALID_ARG):
    return CgvError(code, msg)


def _need_matrix(t, name):
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
        raise _bad(f"{name} must be a CUDA tensor (there is no CPU fallback)")
    if t.dim() != 2:
        raise _bad(f"{name} must be a matrix, got shape {tuple(t.shape)}", CGV_ERR_DIM_MISMATCH)


def _matrix(t, name):
    """A CUDA matrix of a supported type whose rows are contiguous."""
    _need_matrix(t, name)
    if t.dtype not in _CODES:
        raise _bad(f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    if not 1 <= t.shape[1] <= 8192:
        raise _bad(f"{name}: dim must be in 1..=8192, got {t.shape[1]}")
    refuse_tangent(t, name)
    if not t.is_contiguous() and (t.shape[0] <= 1 or t.stride(1) != 1 or t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _ids(t, name, device):
    if not isinstance(t, torch.Tensor) or t.device != device:
        raise _bad(f"{name} must be a tensor on {device}")
    if t.dtype not in (torch.int64, torch.int32):
        raise _bad(f"{name} must be int64 or int32, not {t.dtype}")
    return t if t.dtype == torch.int64 and t.is_contiguous() else t.to(torch.int64).contiguous()


def _workspace(nbytes, device):
    return torch.empty((nbytes,), dtype=torch.uint8, device=device) if nbytes else None


def _lookup(table, ids, scale):
    n, d = table.shape
    dev, k = table.device, ids.numel()
    out = torch.empty((*ids.shape, d), dtype=table.dtype, device=dev)
    _check(lib().cgv_lookup_rows_dev(dev.index, table.data_ptr(), _CODES[table.dtype], n, d, _row_stride(table), ids.data_ptr(), k, scale,
                                     out.data_ptr(), _stream(dev.index)))
    return out


class _LookupRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale):
        ctx.save_for_backward(ids)
        ctx.n, ctx.scale = table.shape[0], scale
        return _lookup(table, ids, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        refuse_tangent(dout, "dout")
        (ids,) = ctx.saved_tensors
        return _lookup_grad(dout.contiguous(), ids, ctx.n, ctx.scale), None, None


def _lookup_grad(dout, ids, n, scale):
    d, k, dev, L = dout.shape[-1], ids.numel(), dout.device, lib()
    out = torch.empty((n, d), dtype=dout.dtype, device=dev)
    nbytes = L.cgv_lookup_grad_workspace(k, n, d)
    ws = _workspace(nbytes, dev)
    _check(L.cgv_lookup_grad_dev(dev.index, dout.data_ptr(), _CODES[dout.dtype], ids.data_ptr(), k, n, d, scale, out.data_ptr(), _ptr(ws), nbytes,
                                 _stream(dev.index)))
    return out


def lookup_rows(table, ids, scale=1.0):
    """scale * table[ids], rounded once to the table's type: ids of any shape (int64 / int32) -> ids.shape + (dim,). An id outside
    [0, n_rows) - the -1 that pads a short search result among them - gives zeros and takes no part in the gradient.
    Differentiable in `table`; the gradient is dense, in the table's type, each row summed in f32 in a fixed order."""
    table = _matrix(table, "table")
    ids = _ids(ids, "ids", table.device)
    if not (table.requires_grad and torch.is_grad_enabled()):
        return _lookup(table, ids, float(scale))
    return _LookupRows.apply(table, ids, float(scale))


def lookup_rows_grad(dout, ids, n_rows, scale=1.0):
    """The gradient of lookup_rows in its table: [n_rows, dim] in dout's type, from dout [..., dim] and ids of dout's leading shape."""
    if not isinstance(dout, torch.Tensor) or dout.device.type != "cuda":
        raise _bad("dout must be a CUDA tensor (there is no CPU fallback)")
    if dout.dtype not in _CODES:
        raise _bad(f"dout must be float32, bfloat16 or float16, not {dout.dtype}")
    refuse_tangent(dout, "dout")
    ids = _ids(ids, "ids", dout.device)
    if dout.dim() < 1 or tuple(dout.shape[:-1]) != tuple(ids.shape):
        raise _bad(f"dout {tuple(dout.shape)} does not fit ids {tuple(ids.shape)}", CGV_ERR_DIM_MISMATCH)
    if int(n_rows) < 0:
        raise _bad("n_rows must be >= 0")
    return _lookup_grad(dout.detach().contiguous(), ids, int(n_rows), float(scale))


def _loss(queries, rows, ids, scores, scale, teacher_scale):
    L = lib()
    b, d = queries.shape
    n, k = rows.shape[0], 1 if scores is None else ids.shape[1]      # the targets of a cross entropy: lists of one
    code, dev = _CODES[rows.dtype], rows.device
    loss = torch.empty((b,), dtype=torch.float32, device=dev)
    saved = torch.empty((b * (k + 2),), dtype=torch.float64, device=dev)
    nbytes = L.cgv_corpus_loss_workspace(b, n, d, k, code)
    ws = _workspace(nbytes, dev)
    _check(L.cgv_corpus_loss_dev(dev.index, queries.data_ptr(), _row_stride(queries), rows.data_ptr(), _row_stride(rows), code, b, n, d, ids.data_ptr(),
                                 _ptr(scores), k, scale, teacher_scale, loss.data_ptr(), saved.data_ptr(), _ptr(ws), nbytes, _stream(dev.index)))
    return loss, saved


class _CorpusLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, queries, rows, ids, scores, scale, teacher_scale):
        loss, saved = _loss(queries, rows, ids, scores, scale, teacher_scale)
        ctx.save_for_backward(queries, rows, ids, scores, saved)
        ctx.scales = (scale, teacher_scale)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        refuse_tangent(dloss, "dloss")
        L = lib()
        queries, rows, ids, scores, saved = ctx.saved_tensors
        b, d = queries.shape
        n, k = rows.shape[0], 1 if scores is None else ids.shape[1]
        code, dev = _CODES[rows.dtype], rows.device
        dq = torch.empty((b, d), dtype=queries.dtype, device=dev) if ctx.needs_input_grad[0] else None
        dr = torch.empty((n, d), dtype=rows.dtype, device=dev) if ctx.needs_input_grad[1] else None
        dloss = dloss.contiguous()
        nbytes = L.cgv_corpus_loss_grad_workspace(b, n, d, k, code)
        ws = _workspace(nbytes, dev)
        _check(L.cgv_corpus_loss_grad_dev(dev.index, _ptr(queries), _row_stride(queries), _ptr(rows), _row_stride(rows), code, b, n, d, _ptr(ids),
                                          _ptr(scores), k, *ctx.scales, _ptr(saved), _ptr(dloss), _ptr(dq), _ptr(dr), _ptr(ws), nbytes,
                                          _stream(dev.index)))
        return dq, dr, None, None, None, None


def _corpus_loss(queries, rows, ids, scores, scale, teacher_scale):
    queries, rows = _matrix(queries, "queries"), _matrix(rows, "rows")
    if queries.device != rows.device:
        raise _bad(f"queries are on {queries.device}, rows on {rows.device}")
    if queries.dtype != rows.dtype:
        raise _bad(f"queries are {queries.dtype}, rows {rows.dtype}")
    if queries.shape[1] != rows.shape[1]:
        raise _bad(f"query dim {queries.shape[1]} != row dim {rows.shape[1]}", CGV_ERR_DIM_MISMATCH)
    if rows.shape[0] == 0:
        raise _bad("rows must not be empty")
    if rows.dtype != torch.float32 and rows.shape[1] % 8 == 0 and (rows.data_ptr() % 16 or _row_stride(rows) % 8 or _row_stride(rows) > 1 << 22):
        rows = rows.clone(memory_format=torch.contiguous_format)      # such rows are read in place, 16 bytes at a time
    if not ((queries.requires_grad or rows.requires_grad) and torch.is_grad_enabled()):
        return _loss(queries, rows, ids, scores, float(scale), float(teacher_scale))[0]
    return _CorpusLoss.apply(queries, rows, ids, scores, float(scale), float(teacher_scale))


def corpus_cross_entropy(queries, rows, targets, scale=1.0):
    """Softmax cross entropy of queries [b, dim] over ALL rows [n, dim] of a corpus: loss[i] = log(sum over j of
    exp(scale * <q_i, r_j>)) - scale * <q_i, r_targets[i]>, f32 [b]. A target outside [0, n) (-1) takes the query out: loss 0, no
    gradient. The b x n scores are never stored. Differentiable in queries and rows; gradients have their types. For 16-bit types the
    scores' gradient is rounded to the type before it is multiplied (more than 32 queries; its listed entries, the largest, are made
    good): include/cgvec_train.h has the bounds; f32 inputs keep f32's digits throughout.
    16-bit rows whose dim is a multiple of 8 are read in place if they start on 16-byte addresses, a multiple of 8 elements (at most 2^22)
    apart; other such rows are copied whole on every call."""
    _need_matrix(queries, "queries")
    targets = _ids(targets, "targets", queries.device)
    if targets.dim() != 1 or targets.shape[0] != queries.shape[0]:
        raise _bad(f"targets {tuple(targets.shape)} do not fit queries {tuple(queries.shape)}", CGV_ERR_DIM_MISMATCH)
    return _corpus_loss(queries, rows, targets, None, scale, 1.0)


def corpus_distillation(queries, rows, teacher_ids, teacher_scores, scale=1.0, teacher_scale=1.0):
    """KL divergence, f32 [b], of softmax(scale * queries @ rows.T) over the WHOLE corpus from the teacher's distribution on its
    list: softmax(teacher_scale * teacher_scores[i]) over the rows teacher_ids[i] ([b, k] each, k <= 256) - the ids and scores
    that a search returns, its padding (-1, -inf) included: entries with an id outside [0, n) or a score of -inf have no weight, a
    query without entries no loss and no gradient. Differentiable in queries and rows; teacher_scores get no gradient.
    Roundings and copies as in corpus_cross_entropy."""
    _need_matrix(queries, "queries")
    ids = _ids(teacher_ids, "teacher_ids", queries.device)
    if not isinstance(teacher_scores, torch.Tensor) or teacher_scores.device != ids.device or not teacher_scores.dtype.is_floating_point:
        raise _bad(f"teacher_scores must be a floating-point tensor on {ids.device}")
    if ids.dim() != 2 or ids.shape[0] != queries.shape[0] or ids.shape != teacher_scores.shape:
        raise _bad(f"teacher_ids {tuple(ids.shape)} and teacher_scores {tuple(teacher_scores.shape)} do not fit queries {tuple(queries.shape)}",
                   CGV_ERR_DIM_MISMATCH)
    refuse_tangent(teacher_scores, "teacher_scores")
    if not 1 <= ids.shape[1] <= 256:
        raise _bad(f"teacher lists must have 1..256 entries, got {ids.shape[1]}")
    return _corpus_loss(queries, rows, ids, teacher_scores.detach().to(torch.float32).contiguous(), scale, teacher_scale)
