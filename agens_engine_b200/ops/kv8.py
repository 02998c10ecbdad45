"""Launchers of the 8-bit key-value cache (``csrc/kernels/sm100/kv8_store.cu``, ``kv8_attn.cu``).

A layer's pool is uint8 ``[pages, hkv, 32 * hd + 128]``: of every page (16 tokens) and KV head the K codes ``[16][hd]``, the V
codes ``[16][hd]`` and sixteen pairs of fp32 scales (K, V).  Formats: ``"int8"`` (codes -127 .. 127, stored with 128 added,
scale = amax / 127 of the row) and ``"fp8"`` (e4m3, scale = amax / 448); a row is one token of one KV head.  A row stands for
code * scale.  Pages and block tables are those of the bf16 pool, at 32 * hd + 128 bytes a page and head instead of
64 * hd.  Reference: the INT8 KV of its dense layers (``kernels/m1/m1_dense8.cu:65-126``, ``kernels/src/kv_tier.cu:32-86``).

Every call runs on the current stream of its tensors' device and can be captured into a CUDA graph.  Index tensors are int32.
What a kernel finds out of range (a page, a position past the block table) sets the ``status`` word to 4 and is skipped.
"""
from __future__ import annotations

import functools
import math
from typing import Optional

import torch

from .. import _lib
from .._lib import Kv8AttnArgs, Kv8ReadArgs, Kv8StoreArgs, check, packer

PAGE = 16
FORMATS = {"int8": 0, "fp8": 1}
GROUP_ROWS = 32                    # most rows of one attention group (bits of a tree mask)
MAX_SPLIT = 2048                   # most keys of one split


def block_bytes(hd: int) -> int:
    """Bytes of one page of one KV head."""
    return 2 * PAGE * hd + 8 * PAGE


def make_pool(n_pages: int, hkv: int, hd: int, device) -> torch.Tensor:
    """An empty pool (zeros) for ``n_pages`` pages."""
    if hd not in (64, 128):
        raise ValueError(f"8-bit KV pages: head_dim 64 or 128, got {hd}")
    return torch.zeros(n_pages, hkv, block_bytes(hd), dtype=torch.uint8, device=device)


@functools.lru_cache(maxsize=256)
def split_keys_for(max_ctx: int, heads: int = 8) -> int:
    """Keys of one attention split for ``heads`` pairs of a sequence and a KV head with contexts of up to ``max_ctx`` tokens: the least of
    128, 256, 512 that makes no more splits than CTAs run at once, else 768, and more where a context had over 256 of them.  A
    constant of the engine, since a row's bits depend on it.

    Small splits spread a short context over the GPU (700 tokens, 8 KV heads: 7.3 us with 128, 8.3 with 256, 9.9 with 512), large ones cost
    less between their keys: 24 sequences of 2000 to 4001 34.7 us with 768, 36.1 with 512, 40.0 with 1024; 131072 tokens 57.1, 57.9, 58.2;
    verify blocks of 4 x 6 rows at 5626 to 9001 51.0, 51.0, 49.2."""
    s = next((s for s in (128, 256, 512) if heads * -(-max_ctx // s) <= 444), 768)
    return next((t for t in (128, 256, 512, 768, 1024) if t >= s and t * 256 >= max_ctx), MAX_SPLIT)


def part_floats(n_tok: int, hq: int, hd: int, max_ctx: int, split_keys: int) -> int:
    """fp32 entries of the workspace that :func:`attn_decode8` needs for ``n_tok`` rows (0: none).  One workspace serves any number
    of calls one after the other; calls that may run at the same time need one each, captured ones too."""
    splits = -(-max_ctx // split_keys)
    return n_tok * hq * splits * (hd + 2) if splits > 1 else 0


# Launches of a step follow one another every few microseconds, so the checks are written to cost little when they pass: one
# expression per argument, the message made only when it fails.
def _fail(what: str):
    raise ValueError("8-bit KV cache: " + what)


def _format(fmt: str) -> int:
    f = FORMATS.get(fmt) if type(fmt) is str else None
    if f is None:
        raise ValueError(f"8-bit KV format: one of {', '.join(FORMATS)}, got {fmt!r}")
    return f


def _check_pool(pool: torch.Tensor, dev: int):
    """Pages, KV heads, head size and address of a pool."""
    shape, at = pool.shape, pool.data_ptr()
    if not (pool.dtype is _U8 and len(shape) == 3 and pool.is_contiguous() and at % 16 == 0):
        _fail("the pool is a contiguous uint8 tensor [pages, hkv, 32 * hd + 128]")
    pages, hkv, size = shape
    hd = _HD_OF.get(size)
    if not (hd and pages):
        _fail(f"a pool of {tuple(shape)} holds no pages of head_dim 64 or 128")
    if pool.get_device() != dev:
        _fail("all tensors on one device")
    return pages, hkv, hd, at


def _check_heads(pool: torch.Tensor, dev: int, hkv: int, hd: int):
    """Pages and address of a pool for ``hkv`` KV heads of ``hd``."""
    pages, heads, size, at = _check_pool(pool, dev)
    if size != hd or heads != hkv:
        _fail(f"the pool's pages are of {heads} KV heads of {size}")
    return pages, at


def _check_index(t: torch.Tensor, n: int, dev: int, name: str) -> int:
    if not (t.dtype is _I32 and t.numel() >= n and t.is_contiguous() and t.get_device() == dev):
        _fail(f"{name}: contiguous int32 with at least {n} entries on the device of the rows")
    return t.data_ptr()


def _check_rows(t: torch.Tensor, n: int, width: int, dev: int, name: str):
    """Distance of two rows of a bf16 [n, width] tensor, and its address."""
    at = t.data_ptr()
    if not (t.dtype is _BF16 and t.shape == (n, width) and t.get_device() == dev):
        _fail(f"{name}: bf16 [{n}, {width}] on the device of the rows")
    ld, unit = (width, 1) if t.is_contiguous() else t.stride()
    if ld % 8 or at % 16 or unit != 1:
        _fail(f"{name}: rows of unit stride that start on 16-byte boundaries")
    return ld, at


def _check_table(bt: torch.Tensor, dev: int):
    """Sequences, pages of a sequence, distance of two rows and address of a block table."""
    shape = bt.shape
    if not (bt.dtype is _I32 and len(shape) == 2 and bt.get_device() == dev):
        _fail("block_table: int32 [sequences, pages] on the device of the rows")
    seqs, cols = shape
    ld, unit = (cols, 1) if bt.is_contiguous() else bt.stride()
    if cols == 0 or unit != 1:
        _fail("block_table: rows of unit stride, at least one page each")
    return seqs, cols, ld, bt.data_ptr()


_BF16, _I32, _U8, _F32 = torch.bfloat16, torch.int32, torch.uint8, torch.float32
_LOG2E = math.log2(math.e)
_HD_OF = {block_bytes(hd): hd for hd in (64, 128)}
_store_args, _attn_args, _read_args = packer(Kv8StoreArgs), packer(Kv8AttnArgs), packer(Kv8ReadArgs)


def _launch(name: str, dev: int, *args):
    """Calls an entry of the library with the current stream of the tensors' device appended."""
    if dev < 0:
        _fail("tensors on a CUDA device")
    fn = getattr(_lib.cuda_lib(), name)
    if torch._C._cuda_getDevice() == dev:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        check(rc, name)


def rope_kvstore8(qkv: torch.Tensor, hq: int, hkv: int, hd: int, inv_freq: torch.Tensor, tok_pos: torch.Tensor, tok_seq: torch.Tensor,
                  block_table: torch.Tensor, pool: torch.Tensor, fmt: str, q_out: torch.Tensor, rope_pos: Optional[torch.Tensor] = None,
                  rope_pos3: Optional[torch.Tensor] = None, pair_axis: Optional[torch.Tensor] = None,
                  status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotates q and k of the fused rows ``qkv`` (bf16 ``[n, (hq + 2 * hkv) * hd]``), writes q to ``q_out`` (bf16 ``[n, hq * hd]``) and
    quantises k and v into slot ``tok_pos[i]`` of sequence ``tok_seq[i]``.  The 8-bit form of ``basic.rope_kvstore`` and, with
    ``rope_pos3`` (int32 ``[3, n]``) and ``pair_axis`` (uint8 ``[hd / 2]``), of ``basic.rope_kvstore_m``; angles are taken in
    64 bits.  Two rows of a call must not name the same slot, and ``q_out`` does not overlap ``qkv``.  A row without a slot (position -1, a
    page that is not there) is not stored and reported; its q is written.  Returns the status word."""
    f, dev = _format(fmt), qkv.get_device()
    n = qkv.shape[0]
    if hq < 1 or hkv < 1:
        _fail("hq and hkv are positive")
    n_pages, at_pool = _check_heads(pool, dev, hkv, hd)
    ld, at_qkv = _check_rows(qkv, n, (hq + 2 * hkv) * hd, dev, "qkv")
    ldq, at_q = _check_rows(q_out, n, hq * hd, dev, "q_out")
    seqs, cols, bt_ld, at_bt = _check_table(block_table, dev)
    at_pos, at_seq = _check_index(tok_pos, n, dev, "tok_pos"), _check_index(tok_seq, n, dev, "tok_seq")
    at_rope = 0 if rope_pos is None else _check_index(rope_pos, n, dev, "rope_pos")
    if not (inv_freq.dtype is _F32 and inv_freq.numel() == hd // 2 and inv_freq.is_contiguous() and inv_freq.get_device() == dev
            and inv_freq.data_ptr() % 16 == 0):
        _fail(f"inv_freq: contiguous fp32 [{hd // 2}] on the device of the rows")
    at_rope3 = at_axis = 0
    if rope_pos3 is not None:
        if pair_axis is None or not (pair_axis.dtype is _U8 and pair_axis.numel() == hd // 2 and pair_axis.is_contiguous() and pair_axis.get_device() == dev):
            _fail(f"rope_pos3 goes with pair_axis, uint8 [{hd // 2}]")
        if rope_pos3.shape != (3, n) or rope_pos is not None:
            _fail(f"rope_pos3: int32 [3, {n}], without rope_pos")
        at_rope3, at_axis = _check_index(rope_pos3, 3 * n, dev, "rope_pos3"), pair_axis.data_ptr()
    if status is None:
        status = torch.zeros(1, dtype=_I32, device=qkv.device)
    at_status = _check_index(status, 1, dev, "status")
    if n:
        a = _store_args(at_qkv, ld, n, hq, hkv, inv_freq.data_ptr(), at_pos, at_rope, at_rope3, at_axis, at_seq, seqs, at_bt, bt_ld, cols, at_pool, n_pages,
                        at_q, ldq, at_status)
        _launch("b2_kv8_store", dev, a, hd, f)
    return status


def attn_decode8(q: torch.Tensor, pool: torch.Tensor, fmt: str, block_table: torch.Tensor, grp_tok0: torch.Tensor, grp_cnt: torch.Tensor,
                 tok_pos: torch.Tensor, tok_seq: torch.Tensor, hq: int, hkv: int, hd: int, split_keys: Optional[int] = None,
                 max_ctx: Optional[int] = None, part: Optional[torch.Tensor] = None, tree_mask: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of new rows over 8-bit pages: ``attention.attn_decode`` for a pool of this module.  ``q``: bf16
    ``[n_tok, hq * hd]`` (RoPE applied).  Group ``g`` is the ``grp_cnt[g]`` (at most 32) rows from ``grp_tok0[g]`` on, all of one
    sequence in ascending order of ``tok_pos``, whose K and V are in the pool already; row i sees the slots up to ``tok_pos[i]``, of
    the slots from the group's first on those whose bit its ``tree_mask`` (int32 ``[n_tok]``) has.  A row that sees nothing
    (``tok_pos`` -1 in a group of its own, an empty mask) gives zeros; rows of no group are left as they were in ``out``, which does
    not overlap ``q``.  Rows of K and V may be as large as 2^100: scores and weights are fp32 numbers.

    ``split_keys`` (a multiple of 16, at most 2048; default :func:`split_keys_for` the table's size) cuts every sequence into
    splits that are joined at the end; a row's bits depend on its own position and on ``split_keys`` only.  ``max_ctx`` (default:
    the table's length) bounds the positions, ``part`` is a workspace of :func:`part_floats` entries (default: allocated for the
    call).  Returns bf16 ``[n_tok, hq * hd]``."""
    f, dev = _format(fmt), q.get_device()
    n = q.shape[0]
    if hkv < 1 or hq < 1 or hq % hkv:
        _fail("hq is a multiple of hkv")
    n_pages, at_pool = _check_heads(pool, dev, hkv, hd)
    ldq, at_q = _check_rows(q, n, hq * hd, dev, "q")
    seqs, cols, bt_ld, at_bt = _check_table(block_table, dev)
    n_groups = grp_tok0.numel()
    at_tok0, at_cnt = _check_index(grp_tok0, n_groups, dev, "grp_tok0"), _check_index(grp_cnt, n_groups, dev, "grp_cnt")
    at_pos, at_seq = _check_index(tok_pos, n, dev, "tok_pos"), _check_index(tok_seq, n, dev, "tok_seq")
    at_mask = 0 if tree_mask is None else _check_index(tree_mask, n, dev, "tree_mask")
    if out is None:
        out = torch.empty(n, hq * hd, dtype=_BF16, device=q.device)
    ldo, at_out = _check_rows(out, n, hq * hd, dev, "out")
    if max_ctx is None:
        max_ctx = cols * PAGE
    elif not 0 < max_ctx <= cols * PAGE:
        _fail(f"max_ctx: 1 .. {cols * PAGE}, what the block table holds")
    if split_keys is None:
        split_keys = split_keys_for(max_ctx, seqs * hkv)
    elif not PAGE <= split_keys <= MAX_SPLIT or split_keys % PAGE:
        _fail(f"split_keys: a multiple of {PAGE} up to {MAX_SPLIT}")
    splits = -(-max_ctx // split_keys)
    slots = n * hq * splits if splits > 1 else 0
    if part is not None and not (part.dtype is _F32 and part.is_contiguous() and part.numel() >= slots * (hd + 2) and part.get_device() == dev
                                 and part.data_ptr() % 16 == 0):
        _fail(f"part: contiguous fp32 with at least {slots * (hd + 2)} entries on the device of the rows")
    if status is None:
        status = torch.zeros(1, dtype=_I32, device=q.device)
    at_status = _check_index(status, 1, dev, "status")
    if n and n_groups:
        if part is None and slots:
            part = torch.empty(slots * (hd + 2), dtype=_F32, device=q.device)
        at_o = part.data_ptr() if slots else 0
        a = _attn_args(at_q, ldq, at_pool, n_pages, at_bt, bt_ld, cols, seqs, at_tok0, at_cnt, n_groups, at_pos, at_seq, n, at_mask, hq, hkv,
                       _LOG2E / math.sqrt(hd), at_out, ldo, at_status, split_keys, splits, at_o, at_o + 4 * slots * hd)
        _launch("b2_kv8_attn", dev, a, hd, f)
    return out


def kv_read8(pool: torch.Tensor, fmt: str, pages: torch.Tensor, n_tokens: Optional[int] = None, out: Optional[torch.Tensor] = None,
             status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The named pages (int32 ``[n]``, a row of a block table or any list) as bf16 pages ``[n, 2, hkv, 16, hd]``, the layout of the
    bf16 pool.  Slots from ``n_tokens`` on (counted over the list) are zeros and are not read; default: every slot."""
    f, dev = _format(fmt), pool.get_device()
    n_pages, hkv, hd, at_pool = _check_pool(pool, dev)
    n = pages.numel()
    at_pages = _check_index(pages, n, dev, "pages")
    if n_tokens is None:
        n_tokens = n * PAGE
    elif not 0 <= n_tokens <= n * PAGE:
        _fail(f"n_tokens: 0 .. {n * PAGE}")
    if out is None:
        out = torch.empty(n, 2, hkv, PAGE, hd, dtype=_BF16, device=pool.device)
    elif not (out.dtype is _BF16 and out.shape == (n, 2, hkv, PAGE, hd) and out.is_contiguous() and out.get_device() == dev and out.data_ptr() % 16 == 0):
        _fail(f"out: contiguous bf16 {[n, 2, hkv, PAGE, hd]} on the device of the pool")
    if status is None:
        status = torch.zeros(1, dtype=_I32, device=pool.device)
    at_status = _check_index(status, 1, dev, "status")
    if n:
        _launch("b2_kv8_read", dev, _read_args(at_pool, n_pages, hkv, at_pages, n, n_tokens, out.data_ptr(), at_status), hd, f)
    return out
