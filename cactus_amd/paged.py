"""ctypes view of the paged INT8 key/value cache (include/cactus_hip_paged.h) for torch device tensors.

A cache is the tuple (k, v, k_scales, v_scales): int8 [num_pages, kv_heads, page_size, head_dim] twice and float32
[num_pages, kv_heads] twice (empty_pages makes one).  block_tables int32 [batch, width] name the pages of each
sequence, and rows of several sequences are packed one behind the other (cu_seqlens int32 [batch + 1]; None: one row
each).  Rows behind the last sequence (a padded batch) are not written: without an output tensor of the caller's they hold
whatever the memory held.  Every function enqueues on torch's current stream of the tensors' device and returns without synchronising.
"""
import ctypes as C

import torch

from . import hip as H

_sz, _vp, _i, _f = C.c_size_t, C.c_void_p, C.c_int, C.c_float


class _PagedKv(C.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("k_scales", _vp), ("v_scales", _vp), ("num_pages", _sz), ("page_size", _sz),
                ("kv_heads", _sz), ("head_dim", _sz)]


PAGED_SIGNATURES = {
    "cactus_hip_kv_append_paged_f16_dev": (_i, [_vp, _vp, _sz, _vp, _vp, _sz, _sz, _vp, _sz, _vp, _sz, _vp, _sz, _vp, _sz,
                                                _vp, _vp, _f, _f, _vp]),
    "cactus_hip_kv_read_paged_f16_dev": (_i, [_vp, _vp, _sz, _vp, _vp, _sz, _sz, _vp, _vp, _vp]),
    "cactus_hip_attention_paged_workspace_bytes": (_sz, [_vp, _sz, _sz, _sz, _sz, _sz, _sz, _i]),
    "cactus_hip_attention_paged_f16_dev": (_i, [_vp, _vp, _sz, _vp, _vp, _sz, _sz, _sz, _vp, _sz, _vp, _sz, _f, _sz, _sz,
                                                _vp, _sz, _vp]),
    "cactus_hip_attention_ragged_f16_dev": (_i, [_vp, _sz, _vp, _sz, _vp, _sz, _vp, _vp, _sz, _sz, _sz, _sz, _sz, _f, _sz,
                                                 _sz, _vp]),
}
for _name, (_res, _args) in PAGED_SIGNATURES.items():
    _fn = getattr(H.lib, _name)  # AttributeError here = the library does not export the header's symbol
    _fn.restype = _res
    _fn.argtypes = _args

# the handle of a device's current stream, without a Stream object around it where torch has the call for that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device

_append = H.lib.cactus_hip_kv_append_paged_f16_dev
_read = H.lib.cactus_hip_kv_read_paged_f16_dev
_attend = H.lib.cactus_hip_attention_paged_f16_dev
_attend_bytes = H.lib.cactus_hip_attention_paged_workspace_bytes
_attend_ragged = H.lib.cactus_hip_attention_ragged_f16_dev


def empty_pages(num_pages, kv_heads, head_dim, page_size=64, device="cuda"):
    """The four tensors of a cache.  Their contents need no clearing: a page starts afresh when its first slot is
    written."""
    pages = lambda: torch.zeros((num_pages, kv_heads, page_size, head_dim), dtype=torch.int8, device=device)  # noqa: E731
    scales = lambda: torch.zeros((num_pages, kv_heads), dtype=torch.float32, device=device)  # noqa: E731
    return pages(), pages(), scales(), scales()


# A decode step calls these functions once per layer with a microsecond or two of work for the GPU, so the checks below read
# every attribute once, compare device numbers instead of device objects, and put their words together only to raise.

def _need(ok, what):
    if not ok:
        raise ValueError("paged: " + what)


def _ints(t, dev, shape, what):
    if t.dtype is not torch.int32 or t.get_device() != dev or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"paged: {what} must be contiguous int32 {list(shape)} on cuda:{dev}, got {t.dtype} "
                         f"{list(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(t, dev, shape, what):
    """Address and row stride of fp16 rows [tokens, heads, head_dim]: heads and head_dim contiguous, rows any stride."""
    if t.dtype is not torch.float16 or t.get_device() != dev or t.shape != shape:
        raise ValueError(f"paged: {what} must be float16 {list(shape)} on cuda:{dev}, got {t.dtype} {list(t.shape)} on {t.device}")
    tokens, heads, dim = shape
    stride, by_head, by_dim = t.stride()
    if by_dim != 1 or (heads > 1 and by_head != dim):
        raise ValueError(f"paged: the heads of a row of {what} must be contiguous, got strides {t.stride()}")
    return t.data_ptr(), stride if tokens > 1 else heads * dim


def _output(t, like, dev, shape, what):
    if t is None:
        return like.new_empty(shape) if like.dtype is torch.float16 else like.new_empty(shape, dtype=torch.float16)
    if t.dtype is not torch.float16 or t.get_device() != dev or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"paged: {what} must be contiguous float16 {list(shape)} on cuda:{dev}")
    return t


def _cache(kv, block_tables):
    """(the C description, device number, batch, table width)"""
    k, v, ks, vs = kv
    shape, dev, int8, f32 = k.shape, k.get_device(), torch.int8, torch.float32
    if dev < 0:
        raise ValueError(f"paged: the cache must be on a GPU, not {k.device}")
    if len(shape) != 4 or k.dtype is not int8 or not k.is_contiguous():
        raise ValueError("paged: k pages must be contiguous int8 [pages, kv_heads, page_size, head_dim]")
    if v.shape != shape or v.dtype is not int8 or v.get_device() != dev or not v.is_contiguous():
        raise ValueError("paged: v pages must be like the k pages")
    pages, heads, size, dim = shape
    per_head = (pages, heads)
    if (ks.shape != per_head or vs.shape != per_head or ks.dtype is not f32 or vs.dtype is not f32 or ks.get_device() != dev
            or vs.get_device() != dev or not ks.is_contiguous() or not vs.is_contiguous()):
        raise ValueError("paged: scales must be contiguous float32 [pages, kv_heads] beside the pages")
    table = block_tables.shape
    _need(len(table) == 2, "block_tables must be [batch, width]")
    _ints(block_tables, dev, table, "block_tables")
    return (_PagedKv(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, size, heads, dim), dev, table[0], table[1])


def _call(dev, fn, *args):
    """fn on the device's current stream, with the device current while it runs."""
    if dev == _current_device():
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        H._check(rc)


def kv_append(k, v, kv, block_tables, positions, theta, cu_seqlens=None, q=None, q_weight=None, k_weight=None, eps=1e-6,
              out_q=None):
    """Append the rows k / v fp16 [tokens, kv_heads, head_dim] of a step or prompt chunk to the cache at positions int32
    [batch] (tokens each sequence already has there; negative: the sequence is skipped), with per-head RMS norm (k_weight),
    rotation (theta; 0: none) and quantization in one launch.  A token that outgrows its page's scale raises it, and the page's
    earlier codes are rounded once more (the header says what that costs).  q fp16 [tokens, q_heads, head_dim], when given, is normed
    (q_weight), rotated and returned."""
    c, dev, batch, width = _cache(kv, block_tables)
    tokens = k.shape[0]
    shape = (tokens, c.kv_heads, c.head_dim)
    kp, kst = _rows(k, dev, shape, "k")
    vp, vst = _rows(v, dev, shape, "v")
    pp = _ints(positions, dev, (batch,), "positions")
    cp = None if cu_seqlens is None else _ints(cu_seqlens, dev, (batch + 1,), "cu_seqlens")
    qp = qst = op = 0
    heads = c.kv_heads
    if q is not None:
        _need(q.dim() == 3, "q must be [tokens, q_heads, head_dim]")
        heads = q.shape[1]
        qp, qst = _rows(q, dev, (tokens, heads, c.head_dim), "q")
        out_q = _output(out_q, q, dev, (tokens, heads, c.head_dim), "out_q")
        op = out_q.data_ptr()
    weights = []
    for w, what in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            if w.dtype is not torch.float16 or w.shape != (c.head_dim,) or w.get_device() != dev or not w.is_contiguous():
                raise ValueError(f"paged: {what} must be float16 [head_dim]")
        weights.append(None if w is None else w.data_ptr())
    _call(dev, _append, C.addressof(c), block_tables.data_ptr(), width, pp, cp, batch, tokens, kp, kst, vp, vst, qp, qst, op,
          heads, weights[0], weights[1], eps, theta)
    return out_q if q is not None else None


def kv_read(kv, block_tables, starts, cu_seqlens, rows, out_k=None, out_v=None):
    """Tokens starts[b] .. of every sequence as fp16 (k, v) [rows, kv_heads, head_dim]; cu_seqlens packs the `rows` rows."""
    c, dev, batch, width = _cache(kv, block_tables)
    sp, cp = _ints(starts, dev, (batch,), "starts"), _ints(cu_seqlens, dev, (batch + 1,), "cu_seqlens")
    shape = (rows, c.kv_heads, c.head_dim)
    out_k, out_v = _output(out_k, kv[0], dev, shape, "out_k"), _output(out_v, kv[0], dev, shape, "out_v")
    _call(dev, _read, C.addressof(c), block_tables.data_ptr(), width, sp, cp, batch, rows, out_k.data_ptr(), out_v.data_ptr())
    return out_k, out_v


def attention(q, kv, block_tables, context_lens, cu_seqlens=None, max_context=None, scale=0.0, window=0, sink=0, out=None):
    """Attention of q fp16 [tokens, q_heads, head_dim] over the cache: context_lens int32 [batch] counts a sequence's
    tokens in the cache, this call's included; the rows of a sequence are its last positions.  window > 0: a position sees
    itself, the `window` positions before it and the first `sink` ones.  max_context: an upper bound of context_lens known
    on the host (default: what block_tables can hold); it only decides how the work is split."""
    c, dev, batch, width = _cache(kv, block_tables)
    _need(q.dim() == 3, "q must be [tokens, q_heads, head_dim]")
    tokens, heads, _ = q.shape
    qp, qst = _rows(q, dev, (tokens, heads, c.head_dim), "q")
    xp = _ints(context_lens, dev, (batch,), "context_lens")
    cp = None if cu_seqlens is None else _ints(cu_seqlens, dev, (batch + 1,), "cu_seqlens")
    if max_context is None:
        max_context = width * c.page_size
    _need(max_context >= 0 and window >= 0 and sink >= 0, "max_context, window and sink must not be negative")
    out = _output(out, q, dev, (tokens, heads, c.head_dim), "out")
    at = C.addressof(c)
    need = _attend_bytes(at, batch, tokens, max_context, heads, window, sink, cp is None)
    work = q.new_empty(need, dtype=torch.uint8) if need else None
    _call(dev, _attend, at, block_tables.data_ptr(), width, xp, cp, batch, tokens, max_context, qp, qst, out.data_ptr(),
          heads, scale, window, sink, work.data_ptr() if need else None, need)
    return out


def attention_ragged(q, k, v, cu_seqlens, scale=0.0, window=0, sink=0, out=None):
    """Causal FP16 attention of prompts packed by cu_seqlens int32 [batch + 1]: q [tokens, q_heads, head_dim], k / v
    [tokens, kv_heads, head_dim]; window and sink as in attention."""
    dev = q.get_device()
    if dev < 0:
        raise ValueError(f"paged: q must be on a GPU, not {q.device}")
    _need(q.dim() == 3 and k.dim() == 3, "q, k and v must be [tokens, heads, head_dim]")
    _need(cu_seqlens.dim() == 1 and cu_seqlens.shape[0] >= 1, "cu_seqlens must be [batch + 1]")
    _need(window >= 0 and sink >= 0, "window and sink must not be negative")
    tokens, heads, dim = q.shape
    kv_heads = k.shape[1]
    qp, qst = _rows(q, dev, (tokens, heads, dim), "q")
    kp, kst = _rows(k, dev, (tokens, kv_heads, dim), "k")
    vp, vst = _rows(v, dev, (tokens, kv_heads, dim), "v")
    batch = cu_seqlens.shape[0] - 1
    cp = _ints(cu_seqlens, dev, (batch + 1,), "cu_seqlens")
    out = _output(out, q, dev, (tokens, heads, dim), "out")
    _call(dev, _attend_ragged, qp, qst, kp, kst, vp, vst, out.data_ptr(), cp, batch, tokens, heads, kv_heads, dim, scale,
          window, sink)
    return out
