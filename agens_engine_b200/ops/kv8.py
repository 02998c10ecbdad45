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

import contextlib
import ctypes as C
import math
from typing import Optional

import torch

from .. import _lib
from .._lib import Kv8AttnArgs, Kv8StoreArgs, check, ptr

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


def split_keys_for(max_ctx: int) -> int:
    """Keys of one attention split for contexts of up to ``max_ctx`` tokens: 256, doubled while more than 64 splits were needed.  A
    constant of the engine, since a row's bits depend on it."""
    s = 256
    while s < MAX_SPLIT and s * 64 < max_ctx:
        s *= 2
    return s


def part_floats(n_tok: int, hq: int, hd: int, max_ctx: int, split_keys: Optional[int] = None) -> int:
    """fp32 entries of the workspace that :func:`attn_decode8` needs for ``n_tok`` rows (0: none).  One workspace serves any number
    of calls one after the other; calls that may run at the same time need one each, captured ones too."""
    splits = -(-max_ctx // (split_keys or split_keys_for(max_ctx)))
    return n_tok * hq * splits * (hd + 2) if splits > 1 else 0


def _format(fmt: str) -> int:
    try:
        return FORMATS[fmt]
    except (KeyError, TypeError):
        raise ValueError(f"8-bit KV format: one of {', '.join(FORMATS)}, got {fmt!r}") from None


def _need(ok: bool, what: str):
    if not ok:
        raise ValueError("8-bit KV cache: " + what)


def _check_pool(pool: torch.Tensor, dev, hkv: Optional[int] = None, hd: Optional[int] = None):
    _need(pool.dtype is torch.uint8 and pool.dim() == 3 and pool.is_contiguous() and pool.data_ptr() % 16 == 0,
          "the pool is a contiguous uint8 tensor [pages, hkv, 32 * hd + 128]")
    got = (pool.shape[2] - 8 * PAGE) // (2 * PAGE)
    _need(got in (64, 128) and pool.shape[2] == block_bytes(got) and pool.shape[0] > 0, f"a pool of {tuple(pool.shape)} holds no pages of head_dim 64 or 128")
    _need((hkv is None or pool.shape[1] == hkv) and (hd is None or got == hd), f"the pool's pages are of {pool.shape[1]} KV heads of {got}")
    _need(pool.device == dev, "all tensors on one device")
    return got


def _check_index(t: Optional[torch.Tensor], n: int, dev, name: str):
    if t is not None:
        _need(t.dtype is torch.int32 and t.numel() >= n and t.is_contiguous() and t.device == dev, f"{name}: contiguous int32 with at least {n} entries on {dev}")


def _check_rows(t: torch.Tensor, n: int, width: int, dev, name: str, align: int):
    _need(t.dtype is torch.bfloat16 and t.dim() == 2 and t.shape[0] == n and t.shape[1] == width and t.device == dev, f"{name}: bf16 [{n}, {width}] on {dev}")
    _need((width == 1 or t.stride(1) == 1) and t.stride(0) % align == 0 and t.data_ptr() % (2 * align) == 0,
          f"{name}: rows of unit stride that start on {2 * align}-byte boundaries")


def _check_table(bt: torch.Tensor, dev):
    _need(bt.dtype is torch.int32 and bt.dim() == 2 and bt.shape[1] > 0 and bt.stride(1) == 1 and bt.device == dev, f"block_table: int32 [sequences, pages] on {dev}")


_HERE = contextlib.nullcontext()


def _on(dev):
    """Makes the tensors' device the current one for the launch."""
    if dev.type != "cuda":
        raise ValueError("8-bit KV cache: tensors on a CUDA device")
    return _HERE if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _status(status: Optional[torch.Tensor], dev) -> torch.Tensor:
    if status is None:
        return torch.zeros(1, dtype=torch.int32, device=dev)
    _check_index(status, 1, dev, "status")
    return status


def rope_kvstore8(qkv: torch.Tensor, hq: int, hkv: int, hd: int, inv_freq: torch.Tensor, tok_pos: torch.Tensor, tok_seq: torch.Tensor,
                  block_table: torch.Tensor, pool: torch.Tensor, fmt: str, q_out: torch.Tensor, rope_pos: Optional[torch.Tensor] = None,
                  rope_pos3: Optional[torch.Tensor] = None, pair_axis: Optional[torch.Tensor] = None,
                  status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotates q and k of the fused rows ``qkv`` (bf16 ``[n, (hq + 2 * hkv) * hd]``), writes q to ``q_out`` (bf16 ``[n, hq * hd]``) and
    quantises k and v into slot ``tok_pos[i]`` of sequence ``tok_seq[i]``.  The 8-bit form of ``basic.rope_kvstore`` and, with
    ``rope_pos3`` (int32 ``[3, n]``) and ``pair_axis`` (uint8 ``[hd / 2]``), of ``basic.rope_kvstore_m``; angles are taken in
    64 bits.  Two rows of a call must not name the same slot.  Returns the status word."""
    f, dev = _format(fmt), qkv.device
    n = qkv.shape[0]
    _need(hq > 0 and hkv > 0, "hq and hkv are positive")
    _check_pool(pool, dev, hkv, hd)
    _check_rows(qkv, n, (hq + 2 * hkv) * hd, dev, "qkv", 4)
    _check_rows(q_out, n, hq * hd, dev, "q_out", 4)
    _check_table(block_table, dev)
    for t, name in ((tok_pos, "tok_pos"), (tok_seq, "tok_seq"), (rope_pos, "rope_pos")):
        _check_index(t, n, dev, name)
    _need(inv_freq.dtype is torch.float32 and inv_freq.numel() == hd // 2 and inv_freq.is_contiguous() and inv_freq.device == dev
          and inv_freq.data_ptr() % 16 == 0, f"inv_freq: fp32 [{hd // 2}]")
    if rope_pos3 is not None:
        _need(pair_axis is not None and pair_axis.dtype is torch.uint8 and pair_axis.numel() == hd // 2 and pair_axis.is_contiguous() and pair_axis.device == dev,
              f"rope_pos3 goes with pair_axis, uint8 [{hd // 2}]")
        _need(tuple(rope_pos3.shape) == (3, n) and rope_pos is None, f"rope_pos3: int32 [3, {n}], without rope_pos")
        _check_index(rope_pos3, 3 * n, dev, "rope_pos3")
    status = _status(status, dev)
    if n == 0:
        return status
    a = Kv8StoreArgs(ptr(qkv), qkv.stride(0), n, hq, hkv, ptr(inv_freq), ptr(tok_pos), ptr(rope_pos), ptr(rope_pos3), ptr(pair_axis), ptr(tok_seq),
                     block_table.shape[0], ptr(block_table), block_table.stride(0), block_table.shape[1], ptr(pool), pool.shape[0], ptr(q_out),
                     q_out.stride(0), ptr(status))
    with _on(dev):
        check(_lib.cuda_lib().b2_kv8_store(C.byref(a), hd, f, torch.cuda.current_stream().cuda_stream), "b2_kv8_store")
    return status


def attn_decode8(q: torch.Tensor, pool: torch.Tensor, fmt: str, block_table: torch.Tensor, grp_tok0: torch.Tensor, grp_cnt: torch.Tensor,
                 tok_pos: torch.Tensor, tok_seq: torch.Tensor, hq: int, hkv: int, hd: int, split_keys: Optional[int] = None,
                 max_ctx: Optional[int] = None, part: Optional[torch.Tensor] = None, tree_mask: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of new rows over 8-bit pages: ``attention.attn_decode`` for a pool of this module.  ``q``: bf16
    ``[n_tok, hq * hd]`` (RoPE applied).  Group ``g`` is the ``grp_cnt[g]`` (at most 32) rows from ``grp_tok0[g]`` on, all of one
    sequence in ascending order of ``tok_pos``, whose K and V are in the pool already; row i sees the slots up to ``tok_pos[i]``, of
    the slots from the group's first on those whose bit its ``tree_mask`` (int32 ``[n_tok]``) has.  A row that sees nothing
    (``tok_pos`` -1 in a group of its own, an empty mask) gives zeros; rows of no group are left as they were in ``out``.

    ``split_keys`` (a multiple of 16, at most 2048; default :func:`split_keys_for` the table's length) cuts every sequence into
    splits that are joined at the end; a row's bits depend on its own position and on ``split_keys`` only.  ``max_ctx`` (default:
    the table's length) bounds the positions, ``part`` is a workspace of :func:`part_floats` entries (default: allocated for the
    call).  Returns bf16 ``[n_tok, hq * hd]``."""
    f, dev = _format(fmt), q.device
    n = q.shape[0]
    _need(hq > 0 and hkv > 0 and hq % hkv == 0, "hq is a multiple of hkv")
    _check_pool(pool, dev, hkv, hd)
    _check_rows(q, n, hq * hd, dev, "q", 8)
    _check_table(block_table, dev)
    n_groups = grp_tok0.numel()
    for t, m, name in ((grp_tok0, n_groups, "grp_tok0"), (grp_cnt, n_groups, "grp_cnt"), (tok_pos, n, "tok_pos"), (tok_seq, n, "tok_seq"), (tree_mask, n, "tree_mask")):
        _check_index(t, m, dev, name)
    if out is None:
        out = torch.empty(n, hq * hd, dtype=torch.bfloat16, device=dev)
    else:
        _check_rows(out, n, hq * hd, dev, "out", 8)
    max_ctx = block_table.shape[1] * PAGE if max_ctx is None else int(max_ctx)
    _need(0 < max_ctx <= block_table.shape[1] * PAGE, f"max_ctx: 1 .. {block_table.shape[1] * PAGE}, what the block table holds")
    split_keys = split_keys_for(max_ctx) if split_keys is None else int(split_keys)
    _need(PAGE <= split_keys <= MAX_SPLIT and split_keys % PAGE == 0, f"split_keys: a multiple of {PAGE} up to {MAX_SPLIT}")
    splits = -(-max_ctx // split_keys)
    slots = n * hq * splits if splits > 1 else 0
    if part is not None:
        _need(part.dtype is torch.float32 and part.is_contiguous() and part.numel() >= slots * (hd + 2) and part.device == dev and part.data_ptr() % 16 == 0,
              f"part: contiguous fp32 with at least {slots * (hd + 2)} entries on {dev}")
    status = _status(status, dev)
    if n == 0 or n_groups == 0:
        return out
    if part is None and slots:
        part = torch.empty(slots * (hd + 2), dtype=torch.float32, device=dev)
    at = ptr(part)
    a = Kv8AttnArgs(ptr(q), q.stride(0), ptr(pool), pool.shape[0], ptr(block_table), block_table.stride(0), block_table.shape[1], block_table.shape[0],
                    ptr(grp_tok0), ptr(grp_cnt), n_groups, ptr(tok_pos), ptr(tok_seq), n, ptr(tree_mask), hq, hkv,
                    math.log2(math.e) / math.sqrt(hd), ptr(out), out.stride(0), ptr(status), split_keys, splits, at, at + 4 * slots * hd)
    with _on(dev):
        check(_lib.cuda_lib().b2_kv8_attn(C.byref(a), hd, f, torch.cuda.current_stream().cuda_stream), "b2_kv8_attn")
    return out


def kv_read8(pool: torch.Tensor, fmt: str, pages: torch.Tensor, n_tokens: Optional[int] = None, out: Optional[torch.Tensor] = None,
             status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The named pages (int32 ``[n]``, a row of a block table or any list) as bf16 pages ``[n, 2, hkv, 16, hd]``, the layout of the
    bf16 pool.  Slots from ``n_tokens`` on (counted over the list) are zeros and are not read; default: every slot."""
    f, dev = _format(fmt), pool.device
    hd = _check_pool(pool, dev)
    n, hkv = pages.numel(), pool.shape[1]
    _check_index(pages, n, dev, "pages")
    n_tokens = n * PAGE if n_tokens is None else int(n_tokens)
    _need(0 <= n_tokens <= n * PAGE, f"n_tokens: 0 .. {n * PAGE}")
    shape = (n, 2, hkv, PAGE, hd)
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    else:
        _need(out.dtype is torch.bfloat16 and tuple(out.shape) == shape and out.is_contiguous() and out.device == dev and out.data_ptr() % 16 == 0, f"out: contiguous bf16 {list(shape)}")
    status = _status(status, dev)
    if n == 0:
        return out
    with _on(dev):
        check(_lib.cuda_lib().b2_kv8_read(ptr(pool), pool.shape[0], hkv, hd, f, ptr(pages), n, n_tokens, ptr(out), ptr(status),
                                          torch.cuda.current_stream().cuda_stream), "b2_kv8_read")
    return out
