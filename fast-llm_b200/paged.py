"""Paged KV cache over the C ABI (``fl_b200_paged_*``): many sequences of unlike length in one pool of pages.

Per step ``plan`` (block tables, slots and positions from the lengths, on the device), per layer ``PagedCache.append`` and
``PagedCache.attn``. Arguments are torch CUDA tensors, checked here for type, shape and device; strides between tokens
are taken from the tensors, so that q, k and v can be slices of one projection's output.

Calls run on the context's stream (``Context.stream``), as everywhere in this library, whatever torch's current stream is. It waits for
torch's default stream and the other way round; work on any other torch stream has to be ordered with it by the caller, by running it
there (``torch.cuda.stream(torch.cuda.ExternalStream(ctx.stream()))``), by events or by ``ctx.sync()``.
"""
import ctypes as C

import torch

from . import capi

F32, F16 = 0, 1
_ACT = {torch.float32: F32, torch.float16: F16}
_I32 = torch.int32
_u32, _p = C.c_uint32, C.c_void_p
_found = {}


class PagedCacheP(C.Structure):
    """Image of fl_b200_paged_cache."""
    _fields_ = [("k_dev", _p), ("v_dev", _p), ("n_pages", _u32), ("page_size", _u32), ("n_kv_head", _u32), ("head_dim", _u32)]


_ARGS = {
    "fl_b200_paged_plan": [_p, _p, _p, _p, _u32, _u32, _p, _u32, _p, _u32, _p, _p, _p, _p, _p, _p, _u32],
    "fl_b200_paged_append": [_p, C.POINTER(PagedCacheP), C.c_int, _p, _u32, _u32, _p, _p, _u32, _p, _p, _u32, _u32, C.c_float, _p, _u32],
    "fl_b200_paged_attn": [_p, C.POINTER(PagedCacheP), C.c_int, _p, _u32, _u32, _p, _u32, _p, _p, _u32, _u32, _u32, C.c_float, _p, _u32, _p],
}


def _entry(lib, name):
    f = _found.get(name)
    if f is None:
        f = getattr(lib, name)
        f.argtypes = _ARGS[name]
        _found[name] = f
    return f


def _ints(dev, name, t, n):
    """Device pointer of a contiguous int32 tensor of n values."""
    if t.dtype is not _I32 or t.numel() != n or not t.is_contiguous() or t.get_device() != dev:
        raise ValueError("%s: a contiguous int32 tensor of %d values on device %d is wanted, got %s %s on %s" % (name, n, dev, t.dtype, tuple(t.shape), t.device))
    return t.data_ptr()


def _fits(name, value):
    """value, which ctypes would cut to 32 bits. (Asked where value >> 32 is not 0.)"""
    if not 0 <= value < 1 << 32:
        raise ValueError("%s: %d is not a 32-bit size" % (name, value))
    return value


def _rows(dev, name, t, dtype, n, width):
    """(pointer, stride) of a 2-D tensor of n tokens whose rows are packed."""
    if t.dtype is not dtype or t.size() != (n, width) or t.get_device() != dev or t.stride(1) != 1:
        raise ValueError("%s: %s activations [%d][%d], packed rows, on device %d are wanted, got %s %s on %s"
                         % (name, dtype, n, width, dev, t.dtype, tuple(t.shape), t.device))
    if n < 2:
        return t.data_ptr(), width
    stride = t.stride(0)
    if stride >> 32:
        _fits(name + "'s stride", stride)
    return t.data_ptr(), stride


def plan(ctx, held, past, new, table, free_list, free_count_in, free_count_out, q_start, kv_len, pos, slot, page_size):
    """fl_b200_paged_plan; table [n_seq][max_blocks], free_list [n_pages], pos and slot [max_tokens]."""
    n_seq, blocks, n_pages, n_tok, dev = held.numel(), table.size(-1), free_list.numel(), pos.numel(), ctx.device
    if page_size >> 32:
        _fits("page_size", page_size)
    capi._ck(_entry(ctx.lib, "fl_b200_paged_plan")(
        ctx._h, _ints(dev, "held", held, n_seq), _ints(dev, "past", past, n_seq), _ints(dev, "new", new, n_seq), n_seq, page_size,
        _ints(dev, "table", table, n_seq * blocks), blocks, _ints(dev, "free_list", free_list, n_pages), n_pages,
        _ints(dev, "free_count_in", free_count_in, 1), _ints(dev, "free_count_out", free_count_out, 1), _ints(dev, "q_start", q_start, n_seq + 1),
        _ints(dev, "kv_len", kv_len, n_seq), _ints(dev, "pos", pos, n_tok), _ints(dev, "slot", slot, n_tok), n_tok))


class PagedCache:
    """K and V pools of one layer ([n_pages][n_kv_head][page_size][head_dim] f16 tensors, which stay the caller's)."""

    def __init__(self, ctx, k, v, n_pages, page_size, n_kv_head, head_dim):
        for name, t in (("k", k), ("v", v)):
            if t.dtype not in (torch.float16, torch.int16) or t.numel() != n_pages * n_kv_head * page_size * head_dim or not t.is_contiguous() \
                    or t.get_device() != ctx.device:
                raise ValueError("%s: a contiguous pool of %d f16 values on device %d is wanted, got %s %s on %s"
                                 % (name, n_pages * n_kv_head * page_size * head_dim, ctx.device, t.dtype, tuple(t.shape), t.device))
        for name, value in (("n_pages", n_pages), ("page_size", page_size), ("n_kv_head", n_kv_head), ("head_dim", head_dim)):
            _fits(name, value)
        self.ctx, self.k, self.v = ctx, k, v
        self.width = n_kv_head * head_dim
        self.cfg = PagedCacheP(k.data_ptr(), v.data_ptr(), n_pages, page_size, n_kv_head, head_dim)

    def append(self, q, k, v, pos, slot, q_out, freq_base, n_rot=None):
        """RoPE on q (into q_out; both None: no q) and k, then k and v into their slots; q, k, v [n_tokens][heads * head_dim]."""
        ctx, dim, width, n, dtype, dev = self.ctx, self.cfg.head_dim, self.width, k.size(0), k.dtype, self.ctx.device
        kp, ks = _rows(dev, "k", k, dtype, n, width)
        vp, vs = _rows(dev, "v", v, dtype, n, width)
        qp, qw, qs, op, os_ = None, 0, 0, None, 0
        if n_rot is None:
            n_rot = dim
        elif n_rot >> 32:
            _fits("n_rot", n_rot)
        if q is not None:
            if q_out is None:
                raise ValueError("append: q goes to q_out")
            qw = q.size(-1)
            qp, qs = _rows(dev, "q", q, dtype, n, qw)
            op, os_ = _rows(dev, "q_out", q_out, dtype, n, qw)
        if dtype not in _ACT or vs != ks or qw % dim:
            raise ValueError("append: f32 or f16 activations of whole heads, k and v of one stride")
        capi._ck(_entry(ctx.lib, "fl_b200_paged_append")(
            ctx._h, self.cfg, _ACT[dtype], qp, qw // dim, qs, kp, vp, ks, _ints(dev, "pos", pos, n), _ints(dev, "slot", slot, n), n,
            n_rot, freq_base, op, os_))

    def attn(self, q, table, q_start, kv_len, max_new, scale, out, lse=None):
        """Causal attention of every sequence's new tokens; q, out [n_tokens][heads * head_dim], lse [n_tokens][heads][2] f32."""
        ctx, dim, n, qw, dtype, dev = self.ctx, self.cfg.head_dim, q.size(0), q.size(-1), q.dtype, self.ctx.device
        n_seq, blocks = kv_len.numel(), table.size(-1)
        if max_new >> 32:
            _fits("max_new", max_new)
        qp, qs = _rows(dev, "q", q, dtype, n, qw)
        op, os_ = _rows(dev, "out", out, dtype, n, qw)
        if dtype not in _ACT or qw % dim:
            raise ValueError("attn: f32 or f16 activations of whole heads")
        if lse is not None and (lse.dtype != torch.float32 or lse.numel() != n * qw // dim * 2 or not lse.is_contiguous() or lse.get_device() != dev):
            raise ValueError("lse: f32 [n_tokens][heads][2] on device %d" % dev)
        capi._ck(_entry(ctx.lib, "fl_b200_paged_attn")(
            ctx._h, self.cfg, _ACT[dtype], qp, qw // dim, qs, _ints(dev, "table", table, n_seq * blocks), blocks,
            _ints(dev, "q_start", q_start, n_seq + 1), _ints(dev, "kv_len", kv_len, n_seq), n_seq, n, max_new, scale, op, os_,
            None if lse is None else lse.data_ptr()))
