"""Torch-facing calls on a paged cache of keys and values: what a verification
round does to the lanes' caches around its decision.

========================  ===========================================================
``norm_rotate_append``     norms and rotation of queries and keys, keys and values
                           written to the lanes' pages
``prefix_attention``       attention of the rows over the pages, a prefix that lanes
                           share read once for all of them
``pages_fork`` / ``pages_extend`` / ``pages_truncate`` / ``pages_compact``
                           who holds which page
``pages_copy`` / ``keep_rows``
                           page contents: whole pages, or the rows of an accepted path
========================  ===========================================================

A cache is one tensor per pool, [..., pages, kv_heads, page_size, head_dim]: the
leading dimensions are the planes (layers, keys and values).  One layer's pages
are views ``pool[layer, 0]`` and ``pool[layer, 1]``.  ``tables`` int32 [lanes,
pages per lane], -1 where a lane holds no page; ``lengths`` int32 [lanes];
``refs`` int32 [pages].  The header of the C ABI has each call's rules.
"""
from __future__ import annotations

import math

import torch

from . import _abi
from ._abi import check
from .ops import _DTYPES, _int_list, _lib, _stream, workspace


def _cache_args(k_pages: torch.Tensor, v_pages: torch.Tensor) -> bytes:
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.stride() != v_pages.stride() or \
            k_pages.dtype != v_pages.dtype:
        raise ValueError("pages must be [pages, kv_heads, page_size, head_dim], keys and values alike")
    if k_pages.stride(3) != 1 or k_pages.dtype not in _DTYPES or not k_pages.is_cuda or not v_pages.is_cuda:
        raise ValueError("pages must be bf16 or fp16 device memory with contiguous head_dim")
    pages, kv_heads, page_size, dim = k_pages.shape
    sp, sh, st, _ = k_pages.stride()
    return _abi.KV_CACHE.pack(k_pages.data_ptr(), v_pages.data_ptr(), sp, sh, st, _DTYPES[k_pages.dtype], pages,
                              page_size, kv_heads, dim, 0)


def _lane_args(tables: torch.Tensor, row_offsets: torch.Tensor, context: torch.Tensor, rows: int) -> bytes:
    if tables.dtype != torch.int32 or tables.dim() != 2 or tables.stride(1) != 1 or not tables.is_cuda:
        raise ValueError("tables must be int32 [lanes, pages per lane] with contiguous rows")
    lanes, width = tables.shape
    return _abi.LANE_ROWS.pack(_int_list(row_offsets, torch.int32, "row_offsets", lanes + 1),
                               _int_list(context, torch.int32, "context", lanes), tables.data_ptr(),
                               max(tables.stride(0), width), width, lanes, rows, 0)


def _head_args(x: torch.Tensor, like: torch.Tensor, rows: int, heads: int, name: str) -> tuple[int, int, int]:
    if x.dim() != 3 or x.dtype != like.dtype or not x.is_cuda or x.stride(2) != 1 or \
            x.shape != (rows, heads, like.shape[3]):
        raise ValueError(f"{name} must be [rows, heads, head_dim] of the pages' type, head_dim contiguous")
    return x.data_ptr(), x.stride(0), x.stride(1)


def norm_rotate_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor,
                       v_pages: torch.Tensor, tables: torch.Tensor, row_offsets: torch.Tensor, context: torch.Tensor,
                       cosines: torch.Tensor | None = None, sines: torch.Tensor | None = None, *,
                       positions: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
                       k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False,
                       out: torch.Tensor | None = None, flags: torch.Tensor | None = None) -> torch.Tensor:
    """Norms and rotation of q [rows, heads, d] and k [rows, kv_heads, d], k and v
    written to the lanes' pages (vi_norm_rotate_append); returns the queries.

    Rows row_offsets[l] .. row_offsets[l + 1] (int32 [lanes + 1]) are lane l's and
    have cache indices from context[l] (int32 [lanes]) on.  cosines / sines: fp32
    [angle rows, rotary / 2] or None (no rotation), row positions[r] (int32
    [rows]; default: the row's cache index).  A weight of None: no norm.  flags:
    int32 [rows], VI_FLAG_ERROR on rows that could not be placed."""
    rows, heads = q.shape[0], q.shape[1]
    cache = _cache_args(k_pages, v_pages)
    kv_heads, dim = k_pages.shape[1], k_pages.shape[3]
    if out is None:
        out = torch.empty(rows, heads, dim, dtype=q.dtype, device=q.device)
    rotary = angle_rows = 0
    if cosines is not None:
        if sines is None or cosines.shape != sines.shape or cosines.dim() != 2 or not cosines.is_contiguous() or \
                not sines.is_contiguous() or cosines.dtype != torch.float32 or sines.dtype != torch.float32 or \
                not cosines.is_cuda or not sines.is_cuda:
            raise ValueError("cosines and sines must be contiguous fp32 [angle rows, rotary / 2] device tensors")
        angle_rows, rotary = cosines.shape[0], 2 * cosines.shape[1]
    elif sines is not None:
        raise ValueError("sines need cosines")
    for w in (q_weight, k_weight):
        if w is not None and (w.dtype != q.dtype or w.shape != (dim,) or not w.is_contiguous() or not w.is_cuda):
            raise ValueError("norm weights must be contiguous [head_dim] of the queries' type")
    qa = _head_args(q, k_pages, rows, heads, "q")
    oa = _head_args(out, k_pages, rows, heads, "out")
    check(_lib().vi_norm_rotate_append(
        cache, _lane_args(tables, row_offsets, context, rows), heads, _abi.HEAD_ROWS.pack(*qa),
        _abi.HEAD_ROWS.pack(*_head_args(k, k_pages, rows, kv_heads, "k")),
        _abi.HEAD_ROWS.pack(*_head_args(v, k_pages, rows, kv_heads, "v")),
        None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), eps,
        _abi.ROTATION.pack(0 if cosines is None else cosines.data_ptr(), 0 if sines is None else sines.data_ptr(),
                           0 if positions is None else _int_list(positions, torch.int32, "positions", rows),
                           angle_rows, rotary, int(interleaved), 0),
        *oa, None if flags is None else _int_list(flags, torch.int32, "flags", rows), _stream()),
        "vi_norm_rotate_append")
    return out


def prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor,
                     row_offsets: torch.Tensor, context: torch.Tensor, *, max_rows: int, max_own: int,
                     group_offsets: torch.Tensor | None = None, prefix_lens: torch.Tensor | None = None,
                     max_group_rows: int = 0, max_prefix: int = 0, tree: torch.Tensor | None = None,
                     scale: float | None = None, out: torch.Tensor | None = None,
                     lse: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q [rows, heads, d] over the lanes' pages (vi_prefix_attention),
    rows, lanes and cache indices as in norm_rotate_append, which has written the
    rows' own keys and values; returns [rows, heads, d].

    group_offsets int32 [groups + 1] / prefix_lens int32 [groups]: lanes that share
    their first tokens, read once for all of a group's rows.  tree: int64 [rows],
    the lane's rows that each row sees (default: those up to itself).  max_rows /
    max_own: bounds of a lane's rows, and of its tokens past the shared prefix;
    max_group_rows / max_prefix: the same of a group.  scale: 1 / sqrt(d) unless
    given.  lse: fp32 [rows, heads], written when given."""
    rows, heads = q.shape[0], q.shape[1]
    cache = _cache_args(k_pages, v_pages)
    kv_heads, dim = k_pages.shape[1], k_pages.shape[3]
    if out is None:
        out = torch.empty(rows, heads, dim, dtype=q.dtype, device=q.device)
    lanes = tables.shape[0]
    groups = go = pl = 0
    if group_offsets is not None:
        if prefix_lens is None:
            raise ValueError("group_offsets need prefix_lens")
        groups = prefix_lens.numel()
        go = _int_list(group_offsets, torch.int32, "group_offsets", groups + 1)
        pl = _int_list(prefix_lens, torch.int32, "prefix_lens")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (rows, heads) or not lse.is_contiguous() or
                            not lse.is_cuda):
        raise ValueError("lse must be contiguous fp32 [rows, heads]")
    qa = _head_args(q, k_pages, rows, heads, "q")
    oa = _head_args(out, k_pages, rows, heads, "out")
    lib, stream = _lib(), _stream()
    nb = lib.vi_prefix_attention_workspace_bytes(rows, heads, kv_heads, dim, lanes, groups, max_rows, max_group_rows,
                                                 max_own, max_prefix)
    ws = workspace(("attention", stream), nb, q.device)
    check(lib.vi_prefix_attention(
        cache, _lane_args(tables, row_offsets, context, rows), heads, _abi.HEAD_ROWS.pack(*qa),
        1.0 / math.sqrt(dim) if scale is None else scale, groups, go, pl, max_rows, max_group_rows, max_own,
        max_prefix, None if tree is None else _int_list(tree, torch.int64, "tree", rows), *oa,
        None if lse is None else lse.data_ptr(), ws.data_ptr(), ws.numel(), stream), "vi_prefix_attention")
    return out


def _map_args(refs: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor | None, page_size: int,
              status: torch.Tensor | None) -> bytes:
    if tables.dtype != torch.int32 or tables.dim() != 2 or tables.stride(1) != 1 or not tables.is_cuda:
        raise ValueError("tables must be int32 [lanes, pages per lane] with contiguous rows")
    lanes, width = tables.shape
    return _abi.PAGE_MAP.pack(_int_list(refs, torch.int32, "refs"), tables.data_ptr(),
                              0 if lengths is None else _int_list(lengths, torch.int32, "lengths", lanes),
                              0 if status is None else _int_list(status, torch.int32, "status", 3),
                              max(tables.stride(0), width), refs.numel(), page_size, lanes, width)


def _pool_args(pool: torch.Tensor, pages: int) -> bytes:
    if pool.dim() < 4 or not pool.is_contiguous() or not pool.is_cuda or pool.shape[-4] != pages:
        raise ValueError("pool must be contiguous [..., pages, kv_heads, page_size, head_dim] device memory")
    page_bytes = pool.stride(-4) * pool.element_size()
    return _abi.PAGE_POOL.pack(pool.data_ptr(), page_bytes * pages, page_bytes, pool.numel() // (pool.stride(-4) * pages),
                               0)


def _pair(a: torch.Tensor, b: torch.Tensor, names: tuple[str, str]) -> tuple[int, int, int]:
    n = a.numel()
    return _int_list(a, torch.int32, names[0]), _int_list(b, torch.int32, names[1], n), n


def pages_fork(refs: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, parents: torch.Tensor,
               children: torch.Tensor, page_size: int, status: torch.Tensor | None = None) -> None:
    """children[i] (int32 lanes) gives back its pages and shares parents[i]'s (vi_pages_fork)."""
    a, b, n = _pair(parents, children, ("parents", "children"))
    check(_lib().vi_pages_fork(_map_args(refs, tables, lengths, page_size, status), a, b, n, _stream()),
          "vi_pages_fork")


def pages_extend(refs: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, lanes: torch.Tensor,
                 new_lengths: torch.Tensor, pool: torch.Tensor, status: torch.Tensor | None = None) -> None:
    """lanes[i] grows to new_lengths[i] tokens, a shared last page copied first
    (vi_pages_extend).  status int32 [3]: flags, pages taken, pages copied."""
    a, b, n = _pair(lanes, new_lengths, ("lanes", "new_lengths"))
    lib, stream = _lib(), _stream()
    ws = workspace(("pages", stream), lib.vi_pages_extend_workspace_bytes(n), refs.device)
    check(lib.vi_pages_extend(_map_args(refs, tables, lengths, pool.shape[-2], status), _pool_args(pool, refs.numel()),
                              a, b, n, ws.data_ptr(), ws.numel(), stream), "vi_pages_extend")


def pages_truncate(refs: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, lanes: torch.Tensor,
                   new_lengths: torch.Tensor, page_size: int, status: torch.Tensor | None = None) -> None:
    """lanes[i] shrinks to new_lengths[i] tokens, 0 frees it (vi_pages_truncate)."""
    a, b, n = _pair(lanes, new_lengths, ("lanes", "new_lengths"))
    check(_lib().vi_pages_truncate(_map_args(refs, tables, lengths, page_size, status), a, b, n, _stream()),
          "vi_pages_truncate")


def pages_copy(pool: torch.Tensor, sources: torch.Tensor, targets: torch.Tensor) -> None:
    """Page sources[i] to page targets[i] in every plane of the pool (vi_pages_copy)."""
    a, b, n = _pair(sources, targets, ("sources", "targets"))
    pages = pool.shape[-4]
    check(_lib().vi_pages_copy(_pool_args(pool, pages), pages, a, b, n, _stream()), "vi_pages_copy")


def pages_compact(refs: torch.Tensor, tables: torch.Tensor, pool: torch.Tensor,
                  status: torch.Tensor | None = None) -> None:
    """The live pages move to the lowest ids (vi_pages_compact).  status int32
    [3]: flags, live pages, pages moved."""
    lib, stream = _lib(), _stream()
    ws = workspace(("pages", stream), lib.vi_pages_compact_workspace_bytes(refs.numel()), refs.device)
    # (a compaction needs no lengths: the tables say what is held)
    check(lib.vi_pages_compact(_map_args(refs, tables, None, pool.shape[-2], status), _pool_args(pool, refs.numel()),
                               ws.data_ptr(), ws.numel(), stream), "vi_pages_compact")


def keep_rows(pool: torch.Tensor, tables: torch.Tensor, lanes: torch.Tensor, context: torch.Tensor,
              paths: torch.Tensor, kept: torch.Tensor) -> None:
    """Row paths[i, j] (int32 [n, width]) of lanes[i], appended at context[i], moves
    to cache index context[i] + j for j < kept[i], in every plane (vi_keep_rows)."""
    n = lanes.numel()
    if paths.dtype != torch.int32 or paths.dim() != 2 or paths.shape[0] != n or not paths.is_contiguous() or \
            not paths.is_cuda:
        raise ValueError("paths must be contiguous int32 [lanes, width] device memory")
    if tables.dtype != torch.int32 or tables.dim() != 2 or tables.stride(1) != 1 or not tables.is_cuda:
        raise ValueError("tables must be int32 [lanes, pages per lane] with contiguous rows")
    pages, kv_heads, page_size, _ = pool.shape[-4:]
    check(_lib().vi_keep_rows(
        _abi.PAGE_MAP.pack(0, tables.data_ptr(), 0, 0, max(tables.stride(0), tables.shape[1]), pages, page_size,
                           tables.shape[0], tables.shape[1]),
        _pool_args(pool, pages), kv_heads, _int_list(lanes, torch.int32, "lanes"),
        _int_list(context, torch.int32, "context", n), paths.data_ptr(), paths.shape[1],
        _int_list(kept, torch.int32, "kept", n), n, _stream()), "vi_keep_rows")
