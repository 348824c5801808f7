"""Paged KV cache over the C ABI (``fl_b200_paged_*``): many sequences of unlike length in one pool of pages.

Per step ``plan`` (block tables, slots and positions from the lengths, on the device), per layer ``PagedCache.append`` and
``PagedCache.attn``. Arguments are torch CUDA tensors, checked here for type, shape and device; strides between tokens
are taken from the tensors, so that q, k and v can be slices of one projection's output.
"""
import ctypes as C

import torch

from . import capi

F32, F16 = 0, 1
_ACT = {torch.float32: F32, torch.float16: F16}
_u32, _p = C.c_uint32, C.c_void_p
_signed = set()


class PagedCacheP(C.Structure):
    """Image of fl_b200_paged_cache."""
    _fields_ = [("k_dev", _p), ("v_dev", _p), ("n_pages", _u32), ("page_size", _u32), ("n_kv_head", _u32), ("head_dim", _u32)]


_ARGS = {
    "fl_b200_paged_plan": [_p, _p, _p, _p, _u32, _u32, _p, _u32, _p, _u32, _p, _p, _p, _p, _p, _p, _u32],
    "fl_b200_paged_append": [_p, C.POINTER(PagedCacheP), C.c_int, _p, _u32, _u32, _p, _p, _u32, _p, _p, _u32, _u32, C.c_float, _p, _u32],
    "fl_b200_paged_attn": [_p, C.POINTER(PagedCacheP), C.c_int, _p, _u32, _u32, _p, _u32, _p, _p, _u32, _u32, _u32, C.c_float, _p, _u32, _p],
}


def _entry(lib, name):
    f = getattr(lib, name)
    if name not in _signed:
        f.argtypes = _ARGS[name]
        _signed.add(name)
    return f


def _ints(ctx, name, t, shape):
    """Device pointer of a contiguous int32 tensor of that shape."""
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous() or t.get_device() != ctx.device:
        raise ValueError("%s: a contiguous int32 tensor %s on device %d is wanted, got %s %s on %s"
                         % (name, tuple(shape), ctx.device, t.dtype, tuple(t.shape), t.device))
    return t.data_ptr()


def _rows(ctx, name, t, act, width=0):
    """(pointer, heads * head_dim, stride) of a 2-D tensor of tokens whose rows are packed."""
    if t.dim() != 2 or t.stride(1) != 1 or t.dtype not in _ACT or _ACT[t.dtype] != act or t.get_device() != ctx.device or (width and t.shape[1] != width):
        raise ValueError("%s: 2-D activations%s of one type, packed rows, on device %d are wanted, got %s %s on %s"
                         % (name, " %d wide" % width if width else "", ctx.device, t.dtype, tuple(t.shape), t.device))
    return t.data_ptr(), t.shape[1], t.stride(0) if t.shape[0] > 1 else t.shape[1]


def plan(ctx, held, past, new, table, free_list, free_count_in, free_count_out, q_start, kv_len, pos, slot, page_size):
    """fl_b200_paged_plan; table [n_seq][max_blocks], free_list [n_pages], pos and slot [max_tokens]."""
    n_seq, blocks, n_pages, n_tok = held.shape[0], table.shape[-1], free_list.shape[0], pos.shape[0]
    capi._ck(_entry(ctx.lib, "fl_b200_paged_plan")(
        ctx._h, _ints(ctx, "held", held, (n_seq,)), _ints(ctx, "past", past, (n_seq,)), _ints(ctx, "new", new, (n_seq,)), n_seq, page_size,
        _ints(ctx, "table", table, (n_seq, blocks)), blocks, _ints(ctx, "free_list", free_list, (n_pages,)), n_pages,
        _ints(ctx, "free_count_in", free_count_in, (1,)), _ints(ctx, "free_count_out", free_count_out, (1,)),
        _ints(ctx, "q_start", q_start, (n_seq + 1,)), _ints(ctx, "kv_len", kv_len, (n_seq,)), _ints(ctx, "pos", pos, (n_tok,)),
        _ints(ctx, "slot", slot, (n_tok,)), n_tok))


class PagedCache:
    """K and V pools of one layer ([n_pages][n_kv_head][page_size][head_dim] f16 tensors, which stay the caller's)."""

    def __init__(self, ctx, k, v, n_pages, page_size, n_kv_head, head_dim):
        for name, t in (("k", k), ("v", v)):
            if t.dtype not in (torch.float16, torch.int16) or t.numel() != n_pages * n_kv_head * page_size * head_dim or not t.is_contiguous() \
                    or t.get_device() != ctx.device:
                raise ValueError("%s: a contiguous pool of %d f16 values on device %d is wanted, got %s %s on %s"
                                 % (name, n_pages * n_kv_head * page_size * head_dim, ctx.device, t.dtype, tuple(t.shape), t.device))
        self.ctx, self.k, self.v = ctx, k, v
        self.cfg = PagedCacheP(k.data_ptr(), v.data_ptr(), n_pages, page_size, n_kv_head, head_dim)

    def append(self, q, k, v, pos, slot, q_out, freq_base, n_rot=None):
        """RoPE on q (into q_out; both None: no q) and k, then k and v into their slots; q, k, v [n_tokens][heads * head_dim]."""
        ctx, cfg, n, act = self.ctx, self.cfg, k.shape[0], _ACT.get(k.dtype)
        width = cfg.n_kv_head * cfg.head_dim
        kp, _, ks = _rows(ctx, "k", k, act, width)
        vp, _, vs = _rows(ctx, "v", v, act, width)
        qp, qw, qs, op, os_ = None, 0, 0, None, 0
        if q is not None:
            qp, qw, qs = _rows(ctx, "q", q, act)
            op, _, os_ = _rows(ctx, "q_out", q_out, act, qw)
        if n > 1 and vs != ks or v.shape[0] != n or qw % cfg.head_dim or (q is not None and (q.shape[0] != n or q_out.shape[0] != n)):
            raise ValueError("append: q, k, v and q_out of one number of tokens and whole heads, k and v of one stride")
        capi._ck(_entry(ctx.lib, "fl_b200_paged_append")(
            ctx._h, self.cfg, act, qp, qw // cfg.head_dim, qs, kp, vp, ks, _ints(ctx, "pos", pos[:n], (n,)), _ints(ctx, "slot", slot[:n], (n,)), n,
            cfg.head_dim if n_rot is None else n_rot, freq_base, op, os_))

    def attn(self, q, table, q_start, kv_len, max_new, scale, out, lse=None):
        """Causal attention of every sequence's new tokens; q, out [n_tokens][heads * head_dim], lse [n_tokens][heads][2] f32."""
        ctx, cfg, act = self.ctx, self.cfg, _ACT.get(q.dtype)
        n, n_seq, blocks = q.shape[0], kv_len.shape[0], table.shape[-1]
        qp, qw, qs = _rows(ctx, "q", q, act)
        op, _, os_ = _rows(ctx, "out", out, act, qw)
        if qw % cfg.head_dim or out.shape[0] != n:
            raise ValueError("attn: whole heads, and an out row for every token")
        if lse is not None and (lse.dtype != torch.float32 or lse.numel() != n * qw // cfg.head_dim * 2 or not lse.is_contiguous() or lse.get_device() != ctx.device):
            raise ValueError("lse: f32 [n_tokens][heads][2]")
        capi._ck(_entry(ctx.lib, "fl_b200_paged_attn")(
            ctx._h, self.cfg, act, qp, qw // cfg.head_dim, qs, _ints(ctx, "table", table, (n_seq, blocks)), blocks,
            _ints(ctx, "q_start", q_start, (n_seq + 1,)), _ints(ctx, "kv_len", kv_len, (n_seq,)), n_seq, n, max_new, scale, op, os_,
            None if lse is None else lse.data_ptr()))
