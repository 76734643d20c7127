"""The paged cache of a continuous batch: append with rotation, decode attention, prompt attention.

The reference pages its cache (KvPages, src/models/inkling/kvpages.rs:1378-1404) and hands attention a list of key runs
(src/models/inkling/flash.rs:995-1015) that all sequences of a call share; `attention.flash_attention_runs` is that
form. Here every sequence has its own pages anywhere in a shared pool, its own length, and both are read on the device,
so a step can be captured into a CUDA graph once and replayed while tables and lengths change.

The order of a step: the host puts the new lengths (this step's tokens included) into `lens`, `paged_append` stores the
rows, `paged_attention_decode` or `paged_attention_prompt` attends. All three work on the current stream of the tensors'
device, which must be the current device.
"""
import ctypes as C
import math
import struct

import torch

from . import _lib
from ._lib import MaryError, lib, context

# A decode step calls these functions once per layer: the checks below are written to cost a microsecond or two, and the
# current stream is asked for without building a Stream object.
_raw_stream = torch._C._cuda_getCurrentRawStream
_bf16_t, _i32_t, _u8_t, _f32_t = torch.bfloat16, torch.int32, torch.uint8, torch.float32
# mb_paged_kv and mb_score_terms as bytes (packing one costs a quarter of building the ctypes structure)
_KV, _TERMS = struct.Struct("@PPPPiNNNNPNNPN"), struct.Struct("@ffNPP")
assert _KV.size == C.sizeof(_lib.PagedKv) and _TERMS.size == C.sizeof(_lib.ScoreTerms)


def _refuse(text):
    raise MaryError(_lib.ERR_INVALID, text)


def _int32(t, name, dims, dev):
    if t.dtype is not _i32_t or t.dim() != dims or t.device != dev:
        _refuse(f"{name} is a {dims}-d int32 tensor on {dev}, not {tuple(t.shape)} {t.dtype} on {t.device}")
    if not t.is_contiguous() and t.stride(dims - 1) != 1:
        _refuse(f"{name} is read with unit stride in its last dimension, not {t.stride()}")


def _ptr(t):
    return t.data_ptr() if t is not None else 0


class PagedCache:
    """Page pools of one layer. bf16 rows: k, v [pages, page_size, kv_heads, head_dim]. NVFP4 rows: k, v code planes
    [pages, page_size, kv_heads * head_dim / 2] uint8 with k_scales, v_scales [pages, page_size, kv_heads * head_dim / 16]
    (the bytes `attention.quantize_kv_rows` gives); head_dim must be told then. head_dim is 64 or 128, page_size a
    multiple of 16. The tensors are used as they are, nothing is copied."""

    def __init__(self, k, v, k_scales=None, v_scales=None, head_dim=None):
        dev = k.device
        if not (k.is_cuda and k.is_contiguous() and v.is_contiguous() and v.device == dev):
            _refuse("page pools are contiguous tensors on one CUDA device")
        if k.shape != v.shape or k.dtype is not v.dtype:
            _refuse(f"k and v pools differ: {tuple(k.shape)} {k.dtype}, {tuple(v.shape)} {v.dtype}")
        if k_scales is None and v_scales is None:
            if k.dtype is not _bf16_t or k.dim() != 4:
                _refuse(f"a pool without scales is [pages, page_size, kv_heads, head_dim] bf16, not {tuple(k.shape)} {k.dtype}")
            self.pages, self.page_size, self.kv_heads, self.head_dim = k.shape
            if head_dim is not None and head_dim != self.head_dim:
                _refuse(f"the pool's head_dim is {self.head_dim}, not {head_dim}")
            self.elem = _lib.KV_BF16
        else:
            if head_dim is None or k_scales is None or v_scales is None:
                _refuse("an NVFP4 pool takes both scale planes and head_dim")
            if k.dtype != torch.uint8 or k.dim() != 3 or head_dim <= 0 or (2 * k.shape[2]) % head_dim:
                _refuse(f"NVFP4 codes are [pages, page_size, kv_heads * {head_dim} / 2] uint8, not {tuple(k.shape)} {k.dtype}")
            for t in (k_scales, v_scales):
                if not t.is_contiguous() or t.device != dev:
                    _refuse("page pools are contiguous tensors on one CUDA device")
                if t.dtype is not _u8_t or tuple(t.shape) != (k.shape[0], k.shape[1], k.shape[2] // 8):
                    _refuse(f"NVFP4 scales of this pool are {(k.shape[0], k.shape[1], k.shape[2] // 8)} uint8, not "
                            f"{tuple(t.shape)} {t.dtype}")
            self.pages, self.page_size, width = k.shape
            self.elem, self.kv_heads, self.head_dim = _lib.KV_NVFP4, 2 * width // head_dim, head_dim
        self.k, self.v, self.k_scales, self.v_scales, self.device = k, v, k_scales, v_scales, dev

    @classmethod
    def empty(cls, pages, page_size, kv_heads, head_dim, nvfp4=False, device=None):
        """Pools without contents (a row is read only after it was appended)."""
        device = device if device is not None else torch.device("cuda", torch.cuda.current_device())
        if not nvfp4:
            make = lambda: torch.empty((pages, page_size, kv_heads, head_dim), dtype=torch.bfloat16, device=device)
            return cls(make(), make())
        width = kv_heads * head_dim
        make = lambda n: torch.empty((pages, page_size, width // n), dtype=torch.uint8, device=device)
        return cls(make(2), make(2), make(16), make(16), head_dim)

    def _kv(self, block_table, lens):
        """(sequences, mb_paged_kv as bytes)"""
        dev = self.device
        _int32(block_table, "block_table", 2, dev)
        _int32(lens, "lens", 1, dev)
        batch, width = block_table.shape
        if lens.shape[0] != batch:
            _refuse(f"block_table has {batch} rows, lens {lens.shape[0]} entries")
        return batch, _KV.pack(self.k.data_ptr(), self.v.data_ptr(), _ptr(self.k_scales), _ptr(self.v_scales), self.elem,
                               self.pages, self.page_size, self.kv_heads, self.head_dim, block_table.data_ptr(), width,
                               block_table.stride(0) if batch > 1 else max(width, 1), lens.data_ptr(), batch)


def _terms(cache, batch, heads, scale, softcap, window, slopes, prefix):
    if slopes is not None and (slopes.dtype is not _f32_t or slopes.shape != (heads,) or not slopes.is_contiguous()
                               or slopes.device != cache.device):
        _refuse(f"slopes is a contiguous f32 tensor of {heads} heads on {cache.device}")
    if prefix is not None:
        _int32(prefix, "prefix", 1, cache.device)
        if prefix.shape[0] != batch:
            _refuse(f"prefix has {prefix.shape[0]} entries for {batch} sequences")
    if window < 0:
        _refuse(f"window is 0 (none) or a positive number of rows, not {window}")
    try:
        return _TERMS.pack(scale if scale is not None else 1.0 / math.sqrt(cache.head_dim), softcap, window, _ptr(slopes),
                           _ptr(prefix))
    except (struct.error, OverflowError, TypeError) as e:
        _refuse(f"scale {scale}, softcap {softcap} and window {window} are two f32 numbers and a count: {e}")


def _bf16(t, name, dev):
    if t.dtype is not _bf16_t or t.device != dev or not t.is_contiguous():
        _refuse(f"{name} is a contiguous bf16 tensor on {dev}")


def _out_like(q, out):
    if out is None:
        return torch.empty_like(q)
    _bf16(out, "out", q.device)
    if out.shape != q.shape:
        _refuse(f"out is {tuple(q.shape)}, not {tuple(out.shape)}")
    return out


def _workspace(workspace, need, dev):
    if need and (workspace is None or workspace.device != dev or workspace.numel() * workspace.element_size() < need
                 or workspace.data_ptr() % 256 or not workspace.is_contiguous()):
        workspace = torch.empty(need, dtype=_u8_t, device=dev)
    return workspace


def paged_append(qkv, cache, block_table, lens, inv_freq, cu_q=None, positions=None, sections=None, out=None):
    """qkv [tokens, (hq + 2 kv_heads) * head_dim] bf16 (rows may be strided): the stacked projection of the batch's new
    tokens. Sequence b's tokens are rows cu_q[b] .. cu_q[b + 1] of it (cu_q [batch + 1] int32 on the device), or, without
    cu_q, an equal share of the rows; they become rows lens[b] - n .. lens[b] of the sequence (lens counts them already).
    q and k heads are rotated by inv_freq [head_dim / 2] f32 at the token's row, or at positions [axes, tokens] int32
    (up to four axes) with `sections` = how many consecutive frequencies follow each axis. Returns the rotated queries
    [tokens, hq, head_dim]; rows at or past cu_q[batch] stay as they are in `out`."""
    dev, d = cache.device, cache.head_dim
    batch, kv = cache._kv(block_table, lens)
    if qkv.dtype is not _bf16_t or qkv.dim() != 2 or qkv.device != dev or qkv.stride(1) != 1:
        _refuse(f"qkv is a 2-d bf16 tensor on {dev} with unit stride along its rows")
    tokens, width = qkv.shape
    hq = width // d - 2 * cache.kv_heads
    if width % d or hq <= 0:
        _refuse(f"a row of {width} values is not (hq + 2 * {cache.kv_heads}) heads of {d}")
    if inv_freq.dtype is not _f32_t or inv_freq.numel() != d // 2 or not inv_freq.is_contiguous() or inv_freq.device != dev:
        _refuse(f"inv_freq is {d // 2} contiguous f32 values on {dev}")
    if cu_q is not None:
        _int32(cu_q, "cu_q", 1, dev)
        if cu_q.shape[0] != batch + 1:
            _refuse(f"cu_q has {cu_q.shape[0]} entries for {batch} sequences")
    axes, ends = 0, None
    if positions is not None:
        if positions.dim() == 1:
            positions = positions.unsqueeze(0)
        _int32(positions, "positions", 2, dev)
        axes = positions.shape[0]
        if positions.shape[1] != tokens or not positions.is_contiguous():
            _refuse(f"positions is contiguous [axes, {tokens}], not {tuple(positions.shape)}")
        sections = (d // 2,) if sections is None and axes == 1 else sections
        if sections is None or len(sections) != axes or sum(sections) != d // 2 or min(sections) < 0:
            _refuse(f"sections are {axes} counts of frequencies that sum to {d // 2}, not {sections}")
        ends = (C.c_int32 * axes)(*[sum(sections[:a + 1]) for a in range(axes)])
    elif sections is not None:
        _refuse("sections belong to positions")
    if out is None:
        out = torch.empty((tokens, hq, d), dtype=_bf16_t, device=dev)
    else:
        _bf16(out, "out", dev)
        if out.numel() != tokens * hq * d:
            _refuse(f"out is [{tokens}, {hq}, {d}], not {tuple(out.shape)}")
    ctx = context(dev.index)
    ctx.check(lib.mb_paged_append(ctx.handle, _raw_stream(dev.index), qkv.data_ptr(), qkv.stride(0) if tokens > 1 else width,
                                  tokens, hq, kv, _ptr(cu_q), inv_freq.data_ptr(), _ptr(positions), axes, ends,
                                  out.data_ptr()))
    return out


def paged_attention_decode(q, cache, block_table, lens, scale=None, softcap=0.0, window=0, slopes=None, prefix=None, out=None,
                           workspace=None):
    """Attention of the last nq tokens of every sequence: q [batch, nq, heads, head_dim] bf16 -> the same shape. Query i of
    sequence b stands at position lens[b] - nq + i; for blocks of eight tokens and more paged_attention_prompt is faster.
    scale: 1 / sqrt(head_dim) by default; softcap, window, slopes [heads] f32 and prefix [batch] int32 as in the header's
    mb_score_terms. A sequence of length 0 gets zeros. workspace: a buffer kept by the caller for calls that do not overlap;
    one is allocated otherwise."""
    _bf16(q, "q", cache.device)
    if q.dim() != 4 or q.shape[3] != cache.head_dim:
        _refuse(f"q is [batch, nq, heads, {cache.head_dim}], not {tuple(q.shape)}")
    batch, kv = cache._kv(block_table, lens)
    q_batch, nq, heads, _ = q.shape
    if q_batch != batch:
        _refuse(f"q has {q_batch} sequences, block_table {batch}")
    terms = _terms(cache, batch, heads, scale, softcap, window, slopes, prefix)
    out = _out_like(q, out)
    ctx = context(cache.device.index)
    need = lib.mb_paged_decode_workspace(ctx.handle, kv, nq, heads)
    workspace = _workspace(workspace, need, cache.device)
    ctx.check(lib.mb_paged_decode(ctx.handle, _raw_stream(ctx.device), q.data_ptr(), nq, heads, kv, terms,
                                  out.data_ptr(), _ptr(workspace), need))
    return out


def paged_attention_prompt(q, cu_q, cache, block_table, lens, scale=None, softcap=0.0, window=0, slopes=None, prefix=None,
                           out=None, workspace=None):
    """Attention of ragged blocks of query tokens: q [tokens, heads, head_dim] bf16, sequence b's are rows cu_q[b] ..
    cu_q[b + 1] (cu_q [batch + 1] int32 on the device) and stand at the sequence's last positions, lens[b] - n .. lens[b].
    Fresh prompts and chunks behind an earlier part alike; no query sees another sequence. The terms and the workspace are
    those of paged_attention_decode; rows at or past cu_q[batch] stay as they are in `out`."""
    _bf16(q, "q", cache.device)
    if q.dim() != 3 or q.shape[2] != cache.head_dim:
        _refuse(f"q is [tokens, heads, {cache.head_dim}], not {tuple(q.shape)}")
    tokens, heads, _ = q.shape
    batch, kv = cache._kv(block_table, lens)
    _int32(cu_q, "cu_q", 1, cache.device)
    if cu_q.shape[0] != batch + 1:
        _refuse(f"cu_q has {cu_q.shape[0]} entries for {batch} sequences")
    terms = _terms(cache, batch, heads, scale, softcap, window, slopes, prefix)
    out = _out_like(q, out)
    ctx = context(cache.device.index)
    need = lib.mb_paged_prompt_workspace(ctx.handle, kv, tokens, heads)
    workspace = _workspace(workspace, need, cache.device)
    ctx.check(lib.mb_paged_prompt(ctx.handle, _raw_stream(ctx.device), q.data_ptr(), tokens, heads, kv, cu_q.data_ptr(),
                                  terms, out.data_ptr(), _ptr(workspace) if need else None, need))
    return out
