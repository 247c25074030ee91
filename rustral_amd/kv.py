"""torch-tensor front end of the paged-KV C ABI.

Device memory and streams come from PyTorch; every computation is one call
into librustral_kv.so on the tensor's current HIP stream.  Pools are
``[num_blocks, Hkv, block_size, D]`` (or ``[n_layers, num_blocks, Hkv,
block_size, D]`` for multi-layer append/copy) in float32 or bfloat16.
"""
from __future__ import annotations

import functools
import math

import torch

from . import _lib
from ._lib import RKV_BF16, RKV_F32, check, lib


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.float32:
        return RKV_F32
    if t.dtype == torch.bfloat16:
        return RKV_BF16
    raise TypeError(f"KV pool dtype {t.dtype}: want float32 or bfloat16")


# The raw handle of a device's current stream without building the Stream object
# (1.7 of a small call's 8 us on the host); a private name, so a torch without it
# takes the public way.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _stream(t: torch.Tensor) -> int:
    return _raw_stream(t.get_device())


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _launch(dev: int, fn, *args) -> None:
    """fn(*args, stream) on device dev's current stream, with dev the current device
    meanwhile: the default stream's handle, 0, means the current device's."""
    if dev == _current_device():
        check(fn(*args, _raw_stream(dev)))
    else:
        with torch.cuda.device(dev):
            check(fn(*args, _raw_stream(dev)))


def _dev(t: torch.Tensor, name: str, dtype=None) -> torch.Tensor:
    if t.is_cuda and (dtype is None or t.dtype is dtype) and t.is_contiguous():
        return t
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _one_device(dev: int, named) -> None:
    """Every tensor on device `dev`: a kernel is launched on one device's stream."""
    for t, name in named:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{name} must be on the call's device")


def _out_like(out: torch.Tensor, q: torch.Tensor) -> torch.Tensor:
    _dev(out, "out", torch.float32)
    if out.shape != q.shape or out.get_device() != q.get_device():
        raise ValueError("out must have q's shape, on its device")
    return out


def check_attention_shapes(q_shape, pool_shape, tables_shape, lens_shape,
                           q_start_shape=None) -> None:
    """The shapes an attention call's kernels index by, checked before any
    launch: q [rows, Hq, D] with D the pool's head_dim and Hq a multiple of
    its KV heads; one block-table row and one length per sequence; q rows one
    per sequence (decode) or q_start of B + 1 offsets (prefill).  The kernels
    take sizes, not buffer lengths, so a mismatch would read past the tables
    or write rows of the wrong width into the pools."""
    hkv, d = pool_shape[1], pool_shape[3]
    if len(q_shape) != 3 or len(tables_shape) != 2 or len(lens_shape) != 1:
        raise ValueError("q, block_tables and ctx_lens must be rank 3, 2 and 1")
    if q_shape[2] != d:
        raise ValueError(f"q head_dim {q_shape[2]} does not match the pool's {d}")
    if q_shape[1] == 0 or q_shape[1] % hkv:
        raise ValueError(f"{q_shape[1]} query heads are not a multiple of {hkv} KV heads")
    seqs = lens_shape[0]
    if tables_shape[0] != seqs:
        raise ValueError(f"{tables_shape[0]} block-table rows for {seqs} sequences")
    if q_start_shape is None:
        if q_shape[0] != seqs:
            raise ValueError(f"{q_shape[0]} q rows for {seqs} sequences")
    elif tuple(q_start_shape) != (seqs + 1,):
        raise ValueError(f"q_start must hold {seqs + 1} offsets")


def append(k_pool: torch.Tensor, v_pool: torch.Tensor, k_new: torch.Tensor,
           v_new: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Scatter new K/V rows into the pools (every layer in one launch).

    k_pool/v_pool: [num_blocks, Hkv, BS, D] or [n_layers, num_blocks, Hkv, BS, D].
    k_new/v_new:   float32 [n_tokens, Hkv, D] or [n_layers, n_tokens, Hkv, D].
    slot_mapping:  int64 [n_tokens], slot = block * BS + row (< 0: skip).
    """
    _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool")
    _dev(k_new, "k_new", torch.float32), _dev(v_new, "v_new", torch.float32)
    _dev(slot_mapping, "slot_mapping", torch.int64)
    multi = k_pool.dim() == 5
    n_layers = k_pool.shape[0] if multi else 1
    nb, hkv, bs, d = k_pool.shape[-4:]
    if k_new.shape != v_new.shape or k_pool.shape != v_pool.shape:
        raise ValueError("K and V shapes differ")
    if k_new.shape[-2:] != (hkv, d) or k_new.dim() != (4 if multi else 3):
        raise ValueError(f"k_new shape {tuple(k_new.shape)} does not match pool {tuple(k_pool.shape)}")
    n_tok = k_new.shape[-3]
    if slot_mapping.shape != (n_tok,):
        raise ValueError("slot_mapping must be [n_tokens]")
    if multi and k_new.shape[0] != n_layers:
        raise ValueError("k_new must have one slice per pool layer")
    pool_ls = nb * hkv * bs * d if multi else 0
    src_ls = n_tok * hkv * d if multi else 0
    check(lib().rkv_append(k_pool.data_ptr(), v_pool.data_ptr(), pool_ls, k_new.data_ptr(),
                           v_new.data_ptr(), src_ls, hkv * d, d, slot_mapping.data_ptr(), n_tok,
                           n_layers, hkv, d, bs, nb, _dtype_code(k_pool), _stream(k_pool)))


def gather(k_pool: torch.Tensor, v_pool: torch.Tensor, block_tables: torch.Tensor,
           ctx_lens: torch.Tensor, *, max_ctx: int | None = None,
           out_offsets: torch.Tensor | None = None, out_total: int | None = None,
           out_dtype: torch.dtype | None = None, k_out=None, v_out=None):
    """Reconstruct contiguous per-sequence K/V (KVCache layout [Hkv, L, D]).

    Padded: returns [B, Hkv, max_ctx, D].  Packed (out_offsets int64 [B] given):
    returns flat tensors of out_total elements.  Untouched rows keep the
    contents of k_out/v_out (zeros when allocated here).
    """
    _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool")
    _dev(block_tables, "block_tables", torch.int32), _dev(ctx_lens, "ctx_lens", torch.int32)
    nb, hkv, bs, d = k_pool.shape
    B, mbs = block_tables.shape
    out_dtype = k_pool.dtype if out_dtype is None else out_dtype
    if out_offsets is None:
        if max_ctx is None:
            max_ctx = mbs * bs
        shape = (B, hkv, max_ctx, d)
        off_ptr = None
    else:
        _dev(out_offsets, "out_offsets", torch.int64)
        if out_total is None:
            raise ValueError("packed gather needs out_total")
        shape = (out_total,)
        off_ptr = out_offsets.data_ptr()
        max_ctx = 0
    if k_out is None:
        k_out = torch.zeros(shape, dtype=out_dtype, device=k_pool.device)
        v_out = torch.zeros(shape, dtype=out_dtype, device=k_pool.device)
    check(lib().rkv_gather(k_out.data_ptr(), v_out.data_ptr(), k_pool.data_ptr(),
                           v_pool.data_ptr(), block_tables.data_ptr(), mbs, ctx_lens.data_ptr(),
                           off_ptr, B, hkv, d, bs, nb, max_ctx, _dtype_code(k_pool),
                           _dtype_code(k_out), _stream(k_pool)))
    return k_out, v_out


def copy_blocks(k_pool: torch.Tensor, v_pool: torch.Tensor, pairs: torch.Tensor) -> None:
    """Block pairs[i,1] := block pairs[i,0] in every layer of the pools.

    pairs: int32 [n_pairs, 2] on the device; destinations must not be sources.
    """
    _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool"), _dev(pairs, "pairs", torch.int32)
    multi = k_pool.dim() == 5
    n_layers = k_pool.shape[0] if multi else 1
    per = k_pool[0] if multi else k_pool
    nb = per.shape[0]
    block_bytes = per[0].numel() * per.element_size()
    layer_stride = per.numel() * per.element_size() if multi else 0
    check(lib().rkv_copy_blocks(k_pool.data_ptr(), v_pool.data_ptr(), layer_stride, n_layers,
                                pairs.data_ptr(), pairs.shape[0], block_bytes, nb,
                                _stream(k_pool)))


# A size is a function of the shape alone: asking the library again costs 0.8 of a
# small call's 8 us on the host.
@functools.lru_cache(maxsize=4096)
def workspace_bytes(num_seqs: int, num_q_heads: int, head_dim: int, max_context: int,
                    partition_size: int = 0) -> int:
    return int(lib().rkv_decode_workspace_bytes(num_seqs, num_q_heads, head_dim, max_context,
                                                partition_size))


def partition_size(dtype_code: int, max_context: int, requested: int = 0, head_dim: int = 128) -> int:
    """The partition size of the split entry points (a request <= 0: 640)."""
    p = lib().rkv_decode_partition_size(requested, head_dim, dtype_code, max_context)
    check(min(p, 0))
    return int(p)


def partition_size_for(num_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                       dtype_code: int, max_context: int, requested: int = 0) -> int:
    """The partition size decode_attention uses for a call of this shape (a
    request <= 0: the library's pick).  With a 1-byte dtype: a size to ask
    decode_attention_q for."""
    p = lib().rkv_decode_partition_size_for(requested, num_seqs, num_q_heads, num_kv_heads,
                                            head_dim, dtype_code, max_context)
    check(min(p, 0))
    return int(p)


def decode_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                     block_tables: torch.Tensor, ctx_lens: torch.Tensor,
                     scale: float | None = None, *, max_context: int | None = None,
                     out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                     passes: str = "both", partition_size: int = 0) -> torch.Tensor:
    """Paged GQA decode attention: q [B, Hq, D] fp32 -> out [B, Hq, D] fp32.

    passes: "both" (default), "partitions" or "merge" (the two launches of
    the split-K algorithm, for callers that time or schedule them apart).
    partition_size: tokens per split-K partition (a multiple of 64 up to
    640, over bf16 pools of 128 up to 1280; 0: partition_size_for's pick).
    """
    _dev(q, "q", torch.float32), _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool")
    _dev(block_tables, "block_tables", torch.int32), _dev(ctx_lens, "ctx_lens", torch.int32)
    nb, hkv, bs, d = k_pool.shape
    check_attention_shapes(q.shape, k_pool.shape, block_tables.shape, ctx_lens.shape)
    B, hq, dq = q.shape
    mbs = block_tables.shape[1]
    if max_context is None:
        max_context = mbs * bs
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.empty_like(q)
    if workspace is None:  # a caller's is checked by the library
        need = workspace_bytes(B, hq, d, max_context, partition_size)
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    ws_ptr = workspace.data_ptr() if workspace is not None else None
    ws_len = workspace.numel() * workspace.element_size() if workspace is not None else 0
    dt = _dtype_code(k_pool)
    s = _stream(q)
    if passes != "both" and partition_size <= 0:
        # the split entry points take 640 for 0: ask for this shape's pick so
        # the two passes partition like the one-call entry point, which goes by
        # the smaller of max_context and the table's tokens and takes 512 where
        # the workspace does not hold a finer pick
        cap = min(max_context, mbs * bs)
        partition_size = partition_size_for(B, hq, hkv, d, dt, cap)
        if partition_size < 512 and ws_len < workspace_bytes(B, hq, d, cap, partition_size):
            partition_size = 512
    if passes in ("both", "partitions"):
        fn = lib().rkv_decode_attention if passes == "both" else lib().rkv_decode_attention_partitions
        check(fn(out.data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
                 block_tables.data_ptr(), mbs, ctx_lens.data_ptr(), B, hq, hkv, d, bs, nb,
                 max_context, float(scale), dt, partition_size, ws_ptr, ws_len, s))
    elif passes == "merge":
        check(lib().rkv_decode_attention_merge(out.data_ptr(), ctx_lens.data_ptr(), mbs, B, hq, d,
                                               bs, max_context, dt, partition_size, ws_ptr, ws_len,
                                               s))
    else:
        raise ValueError(f"passes={passes!r}")
    return out


def decode_attention_append(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                            k_new: torch.Tensor, v_new: torch.Tensor, block_tables: torch.Tensor,
                            ctx_lens: torch.Tensor, scale: float | None = None, *,
                            max_context: int | None = None, out: torch.Tensor | None = None,
                            workspace: torch.Tensor | None = None,
                            partition_size: int = 0) -> torch.Tensor:
    """One decode step's append fused into decode_attention (bf16 pools).

    k_new, v_new: [B, Hkv, D] fp32, the rows of position ctx_lens[b] - 1
    (ctx_lens already counts the new token).  Writes them into the pools and
    returns what append followed by decode_attention returns.
    """
    _dev(q, "q", torch.float32), _dev(k_pool, "k_pool", torch.bfloat16)
    _dev(v_pool, "v_pool", torch.bfloat16)
    _dev(k_new, "k_new", torch.float32), _dev(v_new, "v_new", torch.float32)
    _dev(block_tables, "block_tables", torch.int32), _dev(ctx_lens, "ctx_lens", torch.int32)
    nb, hkv, bs, d = k_pool.shape
    check_attention_shapes(q.shape, k_pool.shape, block_tables.shape, ctx_lens.shape)
    B, hq, dq = q.shape
    if tuple(k_new.shape) != (B, hkv, d) or tuple(v_new.shape) != (B, hkv, d):
        raise ValueError("q, k_new and v_new must be [B, Hq, D], [B, Hkv, D], [B, Hkv, D]")
    mbs = block_tables.shape[1]
    if max_context is None:
        max_context = mbs * bs
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.empty_like(q)
    if workspace is None:  # a caller's is checked by the library
        need = workspace_bytes(B, hq, d, max_context, partition_size)
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    ws_ptr = workspace.data_ptr() if workspace is not None else None
    ws_len = workspace.numel() * workspace.element_size() if workspace is not None else 0
    check(lib().rkv_decode_attention_append(
        out.data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), k_new.data_ptr(),
        v_new.data_ptr(), block_tables.data_ptr(), mbs, ctx_lens.data_ptr(), B, hq, hkv, d, bs,
        nb, max_context, float(scale), _lib.RKV_BF16, partition_size, ws_ptr, ws_len,
        _stream(q)))
    return out


_QFMT = {"int8": _lib.RKV_I8, "fp8": _lib.RKV_FP8, _lib.RKV_I8: _lib.RKV_I8,
         _lib.RKV_FP8: _lib.RKV_FP8}
# one scale a (block, KV head) tile instead of one a row
_BFMT = {"int8_block": _lib.RKV_I8_BLOCK, "fp8_block": _lib.RKV_FP8_BLOCK,
         _lib.RKV_I8_BLOCK: _lib.RKV_I8_BLOCK, _lib.RKV_FP8_BLOCK: _lib.RKV_FP8_BLOCK}
_ANYFMT = {**_QFMT, **_BFMT}


def _qcode(fmt) -> int:
    if fmt not in _QFMT:
        raise ValueError(f"1-byte format {fmt!r}: want 'int8' or 'fp8'")
    return _QFMT[fmt]


def _anycode(fmt) -> int:
    if fmt not in _ANYFMT:
        raise ValueError(f"1-byte format {fmt!r}: want 'int8', 'fp8', 'int8_block' or "
                         "'fp8_block'")
    return _ANYFMT[fmt]


def _bcode(fmt) -> int:
    if fmt not in _BFMT:
        raise ValueError(f"block-scaled format {fmt!r}: want 'int8_block' or 'fp8_block'")
    return _BFMT[fmt]


def _scale_shapes(k_shape, v_shape, ks_shape, vs_shape, code: int) -> None:
    """Scale pools of the shape their format has: one a row, or one a tile.  The
    kernels index them by the byte pools' shape."""
    if v_shape != k_shape:
        raise ValueError("k_pool and v_pool must have one shape")
    cut = -2 if code >= _lib.RKV_I8_BLOCK else -1
    if ks_shape != k_shape[:cut] or vs_shape != v_shape[:cut]:
        raise ValueError("scale pools must be the byte pools' shape without head_dim, and for the "
                         "block formats without the rows too")


def _scale_pools(k_pool, v_pool, k_scale, v_scale, code: int) -> None:
    _dev(k_scale, "k_scale", torch.float32), _dev(v_scale, "v_scale", torch.float32)
    _scale_shapes(k_pool.shape, v_pool.shape, k_scale.shape, v_scale.shape, code)


def _workspace_bytes_q(num_seqs: int, num_q_heads: int, head_dim: int, max_context: int,
                       size: int, fmt) -> int:
    """The workspace of a call over 1-byte pools: row-scaled ones take the split
    entry points' size, not partition_size_for's, where none is asked for."""
    if size <= 0 and fmt in _QFMT:
        size = partition_size(_qcode(fmt), max_context, head_dim=head_dim)
    return workspace_bytes(num_seqs, num_q_heads, head_dim, max_context, size)


def append_q(k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor,
             v_scale: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
             slot_mapping: torch.Tensor, fmt: str = "int8") -> None:
    """Quantizing append into 1-byte pools (uint8 [.., nb, Hkv, BS, D]) with
    per-row fp32 scales ([.., nb, Hkv, BS]); fmt 'int8' or 'fp8' (OCP e4m3)."""
    _dev(k_pool, "k_pool", torch.uint8), _dev(v_pool, "v_pool", torch.uint8)
    _dev(k_scale, "k_scale", torch.float32), _dev(v_scale, "v_scale", torch.float32)
    _dev(k_new, "k_new", torch.float32), _dev(v_new, "v_new", torch.float32)
    _dev(slot_mapping, "slot_mapping", torch.int64)
    multi = k_pool.dim() == 5
    n_layers = k_pool.shape[0] if multi else 1
    nb, hkv, bs, d = k_pool.shape[-4:]
    if k_scale.shape != k_pool.shape[:-1] or v_scale.shape != v_pool.shape[:-1]:
        raise ValueError("scale pools must be the byte pools' shape without head_dim")
    n_tok = k_new.shape[-3]
    if slot_mapping.shape != (n_tok,) or k_new.shape[-2:] != (hkv, d):
        raise ValueError("k_new / slot_mapping shapes do not match the pool")
    pool_ls = nb * hkv * bs * d if multi else 0
    src_ls = n_tok * hkv * d if multi else 0
    check(lib().rkv_append_q(k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr(),
                             v_scale.data_ptr(), pool_ls, k_new.data_ptr(), v_new.data_ptr(),
                             src_ls, hkv * d, d, slot_mapping.data_ptr(), n_tok, n_layers, hkv,
                             d, bs, nb, _qcode(fmt), _stream(k_pool)))


def gather_q(k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor,
             v_scale: torch.Tensor, block_tables: torch.Tensor, ctx_lens: torch.Tensor,
             fmt: str = "int8", *, max_ctx: int | None = None,
             out_offsets: torch.Tensor | None = None, out_total: int | None = None,
             k_out=None, v_out=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Dequantized K/V per sequence in fp32: padded [B, Hkv, max_ctx, D], or
    packed (out_offsets int64 [B] given) as flat tensors of out_total
    elements.  Untouched rows keep the contents of k_out/v_out (zeros when
    allocated here).  Any 1-byte format; the block formats' scale pools are
    [num_blocks, Hkv]."""
    code = _anycode(fmt)
    if code >= _lib.RKV_I8_BLOCK:
        _scale_pools(k_pool, v_pool, k_scale, v_scale, code)
    _dev(k_pool, "k_pool", torch.uint8), _dev(v_pool, "v_pool", torch.uint8)
    _dev(k_scale, "k_scale", torch.float32), _dev(v_scale, "v_scale", torch.float32)
    _dev(block_tables, "block_tables", torch.int32), _dev(ctx_lens, "ctx_lens", torch.int32)
    nb, hkv, bs, d = k_pool.shape
    B, mbs = block_tables.shape
    if out_offsets is None:
        if max_ctx is None:
            max_ctx = mbs * bs
        shape = (B, hkv, max_ctx, d)
        off_ptr = None
    else:
        _dev(out_offsets, "out_offsets", torch.int64)
        if out_total is None:
            raise ValueError("packed gather needs out_total")
        shape = (out_total,)
        off_ptr = out_offsets.data_ptr()
        max_ctx = 0
    if k_out is None:
        k_out = torch.zeros(shape, dtype=torch.float32, device=k_pool.device)
        v_out = torch.zeros(shape, dtype=torch.float32, device=k_pool.device)
    _dev(k_out, "k_out", torch.float32), _dev(v_out, "v_out", torch.float32)
    if k_out.numel() < math.prod(shape) or v_out.numel() < math.prod(shape):
        raise ValueError("gather_q output smaller than the layout needs")
    check(lib().rkv_gather_q(k_out.data_ptr(), v_out.data_ptr(), k_pool.data_ptr(),
                             v_pool.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                             block_tables.data_ptr(), mbs, ctx_lens.data_ptr(), off_ptr, B, hkv, d,
                             bs, nb, max_ctx, code, _stream(k_pool)))
    return k_out, v_out


def decode_attention_append_q(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                              k_scale: torch.Tensor, v_scale: torch.Tensor, k_new: torch.Tensor,
                              v_new: torch.Tensor, block_tables: torch.Tensor,
                              ctx_lens: torch.Tensor, scale: float | None = None,
                              fmt: str = "int8", *, max_context: int | None = None,
                              out: torch.Tensor | None = None,
                              workspace: torch.Tensor | None = None,
                              partition_size: int = 0) -> torch.Tensor:
    """decode_attention_append over 1-byte pools: the new rows quantized as
    append_q quantizes them, then decode_attention_q, in one launch.
    partition_size 0: 640 (see decode_attention_q)."""
    _dev(q, "q", torch.float32), _dev(k_pool, "k_pool", torch.uint8)
    _dev(v_pool, "v_pool", torch.uint8), _dev(k_scale, "k_scale", torch.float32)
    _dev(v_scale, "v_scale", torch.float32)
    _dev(k_new, "k_new", torch.float32), _dev(v_new, "v_new", torch.float32)
    _dev(block_tables, "block_tables", torch.int32), _dev(ctx_lens, "ctx_lens", torch.int32)
    nb, hkv, bs, d = k_pool.shape
    check_attention_shapes(q.shape, k_pool.shape, block_tables.shape, ctx_lens.shape)
    B, hq, dq = q.shape
    if tuple(k_new.shape) != (B, hkv, d) or tuple(v_new.shape) != (B, hkv, d):
        raise ValueError("q, k_new and v_new must be [B, Hq, D], [B, Hkv, D], [B, Hkv, D]")
    mbs = block_tables.shape[1]
    if max_context is None:
        max_context = mbs * bs
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.empty_like(q)
    if workspace is None:  # a caller's is checked by the library
        need = _workspace_bytes_q(B, hq, d, max_context, partition_size, fmt)
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    ws_ptr = workspace.data_ptr() if workspace is not None else None
    ws_len = workspace.numel() * workspace.element_size() if workspace is not None else 0
    check(lib().rkv_decode_attention_append_q(
        out.data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr(),
        v_scale.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), block_tables.data_ptr(), mbs,
        ctx_lens.data_ptr(), B, hq, hkv, d, bs, nb, max_context, float(scale), _qcode(fmt),
        partition_size, ws_ptr, ws_len, _stream(q)))
    return out


def decode_attention_q(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                       k_scale: torch.Tensor, v_scale: torch.Tensor, block_tables: torch.Tensor,
                       ctx_lens: torch.Tensor, scale: float | None = None, fmt: str = "int8", *,
                       max_context: int | None = None, out: torch.Tensor | None = None,
                       workspace: torch.Tensor | None = None, partition_size: int = 0) -> torch.Tensor:
    """decode_attention over 1-byte pools: per-row scales ('int8', 'fp8'), or one
    scale a block and KV head ('int8_block', 'fp8_block').
    partition_size 0: 640 over row-scaled pools, where partition_size_for gives
    the size to ask for if a small call wants finer partitions; its pick over
    block-scaled ones."""
    code = _anycode(fmt)
    u8, f32, i32 = torch.uint8, torch.float32, torch.int32
    dev = q.get_device()
    if not (dev >= 0 and q.dtype is f32 and k_pool.dtype is u8 and v_pool.dtype is u8 and
            k_scale.dtype is f32 and v_scale.dtype is f32 and block_tables.dtype is i32 and
            ctx_lens.dtype is i32 and q.is_contiguous() and k_pool.is_contiguous() and
            v_pool.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous() and
            block_tables.is_contiguous() and ctx_lens.is_contiguous() and
            dev == k_pool.get_device() == v_pool.get_device() == k_scale.get_device() ==
            v_scale.get_device() == block_tables.get_device() == ctx_lens.get_device()):
        _dev(q, "q", f32), _dev(k_pool, "k_pool", u8)  # says which and why
        _dev(v_pool, "v_pool", u8), _dev(k_scale, "k_scale", f32)
        _dev(v_scale, "v_scale", f32)
        _dev(block_tables, "block_tables", i32), _dev(ctx_lens, "ctx_lens", i32)
        _one_device(dev, ((k_pool, "k_pool"), (v_pool, "v_pool"), (k_scale, "k_scale"),
                          (v_scale, "v_scale"), (block_tables, "block_tables"),
                          (ctx_lens, "ctx_lens")))
    shape, tables = k_pool.shape, block_tables.shape
    nb, hkv, bs, d = shape
    if code >= _lib.RKV_I8_BLOCK:
        _scale_shapes(shape, v_pool.shape, k_scale.shape, v_scale.shape, code)
    check_attention_shapes(q.shape, shape, tables, ctx_lens.shape)
    B, hq, _ = q.shape
    mbs = tables[1]
    if max_context is None:
        max_context = mbs * bs
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.empty_like(q)
    if workspace is None:  # a caller's is checked by the library
        need = _workspace_bytes_q(B, hq, d, max_context, partition_size, fmt)
        if need:
            workspace = q.new_empty(need, dtype=torch.uint8)
    ws_ptr = workspace.data_ptr() if workspace is not None else None
    ws_len = workspace.numel() * workspace.element_size() if workspace is not None else 0
    _launch(dev, lib().rkv_decode_attention_q, out.data_ptr(), q.data_ptr(), k_pool.data_ptr(),
            v_pool.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), block_tables.data_ptr(),
            mbs, ctx_lens.data_ptr(), B, hq, hkv, d, bs, nb, max_context, float(scale), code,
            partition_size, ws_ptr, ws_len)
    return out


def prefill_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                      block_tables: torch.Tensor, q_start: torch.Tensor, ctx_lens: torch.Tensor,
                      scale: float | None = None, *, max_q_len: int | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal prefill attention: q [total, Hq, D] fp32 -> out [total, Hq, D].

    Sequence b owns rows q_start[b] .. q_start[b+1]-1 (int32 [B+1]); its new
    tokens are the last ones of its ctx_lens[b] cached tokens (appended
    beforehand).  max_q_len bounds every sequence's new-token count (computed
    from q_start, with a device sync, when not given).
    """
    _dev(q, "q", torch.float32), _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool")
    _dev(block_tables, "block_tables", torch.int32), _dev(ctx_lens, "ctx_lens", torch.int32)
    _dev(q_start, "q_start", torch.int32)
    nb, hkv, bs, d = k_pool.shape
    total, hq, dq = q.shape
    B = ctx_lens.shape[0]
    check_attention_shapes(q.shape, k_pool.shape, block_tables.shape, ctx_lens.shape,
                           q_start.shape)
    if max_q_len is None:
        max_q_len = int((q_start[1:] - q_start[:-1]).max().item()) if B else 0
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.zeros_like(q)
    check(lib().rkv_prefill_attention(out.data_ptr(), q.data_ptr(), k_pool.data_ptr(),
                                      v_pool.data_ptr(), block_tables.data_ptr(),
                                      block_tables.shape[1], q_start.data_ptr(),
                                      ctx_lens.data_ptr(), B, hq, hkv, d, bs, nb, max_q_len,
                                      float(scale), _dtype_code(k_pool), _stream(q)))
    return out


def append_block_q(k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor,
                   v_scale: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                   new_start: torch.Tensor, block_tables: torch.Tensor, ctx_lens: torch.Tensor,
                   fmt: str = "int8_block", *, max_new: int | None = None) -> None:
    """Quantizing append into pools with one scale a (block, KV head) tile:
    uint8 [.., nb, Hkv, 16, D] with fp32 scales [.., nb, Hkv].

    k_new / v_new: float32 [total, Hkv, D] or [n_layers, total, Hkv, D]; sequence
    b's rows are new_start[b] .. new_start[b+1]-1 (int32 [B+1]), the last ones of
    its ctx_lens[b] tokens.  A block's scale grows to hold its new rows, and its
    older rows are rounded to it.  max_new bounds every sequence's row count
    (computed from new_start, with a device sync, when not given).
    """
    code = _bcode(fmt)
    u8, f32, i32 = torch.uint8, torch.float32, torch.int32
    dev = k_pool.get_device()
    if not (dev >= 0 and k_pool.dtype is u8 and v_pool.dtype is u8 and k_scale.dtype is f32 and
            v_scale.dtype is f32 and k_new.dtype is f32 and v_new.dtype is f32 and
            new_start.dtype is i32 and block_tables.dtype is i32 and ctx_lens.dtype is i32 and
            k_pool.is_contiguous() and v_pool.is_contiguous() and k_scale.is_contiguous() and
            v_scale.is_contiguous() and k_new.is_contiguous() and v_new.is_contiguous() and
            new_start.is_contiguous() and block_tables.is_contiguous() and
            ctx_lens.is_contiguous() and
            dev == v_pool.get_device() == k_scale.get_device() == v_scale.get_device() ==
            k_new.get_device() == v_new.get_device() == new_start.get_device() ==
            block_tables.get_device() == ctx_lens.get_device()):
        _dev(k_pool, "k_pool", u8), _dev(v_pool, "v_pool", u8)  # says which and why
        _dev(k_scale, "k_scale", f32), _dev(v_scale, "v_scale", f32)
        _dev(k_new, "k_new", f32), _dev(v_new, "v_new", f32)
        _dev(new_start, "new_start", i32), _dev(block_tables, "block_tables", i32)
        _dev(ctx_lens, "ctx_lens", i32)
        _one_device(dev, ((v_pool, "v_pool"), (k_scale, "k_scale"), (v_scale, "v_scale"),
                          (k_new, "k_new"), (v_new, "v_new"), (new_start, "new_start"),
                          (block_tables, "block_tables"), (ctx_lens, "ctx_lens")))
    shape = k_pool.shape
    multi = len(shape) == 5
    n_layers = shape[0] if multi else 1
    nb, hkv, bs, d = shape[-4:]
    if shape != v_pool.shape or k_new.shape != v_new.shape:
        raise ValueError("K and V shapes differ")
    if k_scale.shape != shape[:-2] or v_scale.shape != shape[:-2]:
        raise ValueError("scale pools must be the byte pools' shape without rows and head_dim")
    *lead, total, rh, rd = k_new.shape
    if rh != hkv or rd != d or lead != ([n_layers] if multi else []):
        raise ValueError(f"k_new shape {tuple(k_new.shape)} does not match pool {tuple(shape)}")
    (B,) = ctx_lens.shape
    rows, mbs = block_tables.shape
    if rows != B or new_start.shape != (B + 1,):
        raise ValueError("one block-table row and one length per sequence, new_start B + 1 offsets")
    if max_new is None:
        max_new = int((new_start[1:] - new_start[:-1]).max().item()) if B else 0
    _launch(dev, lib().rkv_append_block_q, k_pool.data_ptr(), v_pool.data_ptr(),
            k_scale.data_ptr(), v_scale.data_ptr(), nb * hkv * bs * d if multi else 0,
            k_new.data_ptr(), v_new.data_ptr(), total * hkv * d if multi else 0, hkv * d, d,
            new_start.data_ptr(), block_tables.data_ptr(), mbs, ctx_lens.data_ptr(), B, n_layers,
            hkv, d, bs, nb, max_new, code)


def prefill_attention_q(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                        k_scale: torch.Tensor, v_scale: torch.Tensor,
                        block_tables: torch.Tensor, q_start: torch.Tensor,
                        ctx_lens: torch.Tensor, scale: float | None = None,
                        fmt: str = "int8_block", *, max_q_len: int | None = None,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """prefill_attention over block-scaled 8-bit pools ('int8_block',
    'fp8_block')."""
    code = _bcode(fmt)
    u8, f32, i32 = torch.uint8, torch.float32, torch.int32
    dev = q.get_device()
    if not (dev >= 0 and q.dtype is f32 and k_pool.dtype is u8 and v_pool.dtype is u8 and
            k_scale.dtype is f32 and v_scale.dtype is f32 and block_tables.dtype is i32 and
            q_start.dtype is i32 and ctx_lens.dtype is i32 and q.is_contiguous() and
            k_pool.is_contiguous() and v_pool.is_contiguous() and k_scale.is_contiguous() and
            v_scale.is_contiguous() and block_tables.is_contiguous() and
            q_start.is_contiguous() and ctx_lens.is_contiguous() and
            dev == k_pool.get_device() == v_pool.get_device() == k_scale.get_device() ==
            v_scale.get_device() == block_tables.get_device() == q_start.get_device() ==
            ctx_lens.get_device()):
        _dev(q, "q", f32), _dev(k_pool, "k_pool", u8)  # says which and why
        _dev(v_pool, "v_pool", u8), _dev(k_scale, "k_scale", f32)
        _dev(v_scale, "v_scale", f32), _dev(q_start, "q_start", i32)
        _dev(block_tables, "block_tables", i32), _dev(ctx_lens, "ctx_lens", i32)
        _one_device(dev, ((k_pool, "k_pool"), (v_pool, "v_pool"), (k_scale, "k_scale"),
                          (v_scale, "v_scale"), (q_start, "q_start"),
                          (block_tables, "block_tables"), (ctx_lens, "ctx_lens")))
    _scale_shapes(k_pool.shape, v_pool.shape, k_scale.shape, v_scale.shape, code)
    check_attention_shapes(q.shape, k_pool.shape, block_tables.shape, ctx_lens.shape,
                           q_start.shape)
    nb, hkv, bs, d = k_pool.shape
    B = ctx_lens.shape[0]
    if max_q_len is None:
        max_q_len = int((q_start[1:] - q_start[:-1]).max().item()) if B else 0
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.zeros_like(q)
    else:
        _out_like(out, q)
    _launch(dev, lib().rkv_prefill_attention_q, out.data_ptr(), q.data_ptr(),
            k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
            block_tables.data_ptr(), block_tables.shape[1], q_start.data_ptr(),
            ctx_lens.data_ptr(), B, q.shape[1], hkv, d, bs, nb, max_q_len, float(scale), code)
    return out


# ---- rotary positions ----------------------------------------------------------

_ROPE = {None: _lib.RKV_ROPE_PLAIN, "linear": _lib.RKV_ROPE_LINEAR, "base": _lib.RKV_ROPE_BASE,
         "parts": _lib.RKV_ROPE_PARTS, "bands": _lib.RKV_ROPE_BANDS}


def rope_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: str | None = None,
                     factor: float = 1.0, original_context: int = 0, low: float = 1.0,
                     high: float = 32.0, device=None) -> tuple[torch.Tensor, float]:
    """The table and magnitude that rope and rope_append take: float64
    [rotary_dim / 2] on the device, and a float.  scaling: None, 'linear',
    'base', 'parts' or 'bands' (rkv_rope_frequencies says what each does)."""
    if scaling not in _ROPE:
        raise ValueError(f"scaling {scaling!r}: want one of {list(_ROPE)}")
    out = torch.empty(max(rotary_dim // 2, 0), dtype=torch.float64)
    magnitude = torch.empty(1, dtype=torch.float32)
    check(lib().rkv_rope_frequencies(out.data_ptr(), magnitude.data_ptr(), rotary_dim,
                                     float(base), _ROPE[scaling], float(factor),
                                     original_context, float(low), float(high)))
    return out.to(device if device is not None else "cuda"), float(magnitude)


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """fp32 rows [T, H, D] whose elements are contiguous (a slice of a fused
    projection's output is fine)."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be {torch.float32}, got {t.dtype}")
    if t.dim() != 3 or (t.shape[2] > 1 and t.stride(2) != 1):
        raise ValueError(f"{name} must be [tokens, heads, head_dim] with contiguous rows")
    return t


def _rope_tensors(positions: torch.Tensor, inv_freq: torch.Tensor) -> None:
    _dev(positions, "positions", torch.int32), _dev(inv_freq, "inv_freq", torch.float64)


def _rope_shapes(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor) -> None:
    _rope_tensors(positions, inv_freq)
    _one_device(x.get_device(), ((positions, "positions"), (inv_freq, "inv_freq")))
    if positions.shape != (x.shape[0],):
        raise ValueError(f"{tuple(positions.shape)} positions for {x.shape[0]} tokens")
    if inv_freq.dim() != 1 or 2 * inv_freq.shape[0] > x.shape[2]:
        raise ValueError("inv_freq must be [rotary_dim / 2] with rotary_dim <= head_dim")


def rope(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *,
         interleaved: bool = False, magnitude: float = 1.0,
         out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions: rows x [T, H, D] fp32 turned by positions [T] (int32)
    times inv_freq (float64 [rotary_dim / 2], rope_frequencies).  The rotated
    dims are the first rotary_dim, as pairs (i, i + rotary_dim / 2), or (2 i,
    2 i + 1) with interleaved.  out may be x."""
    _rows(x, "x")
    _rope_shapes(x, positions, inv_freq)
    if out is None:
        out = x.new_empty(x.shape)
    elif _rows(out, "out").shape != x.shape or out.get_device() != x.get_device():
        raise ValueError("out must have x's shape, on its device")
    t, h, d = x.shape
    _launch(x.get_device(), lib().rkv_rope, out.data_ptr(), x.data_ptr(), positions.data_ptr(),
            inv_freq.data_ptr(), t, h, d, 2 * inv_freq.shape[0], out.stride(0), out.stride(1),
            x.stride(0), x.stride(1), int(interleaved), magnitude)
    return out


def rope_append(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                positions: torch.Tensor, inv_freq: torch.Tensor, k_pool: torch.Tensor,
                v_pool: torch.Tensor, slot_mapping: torch.Tensor, *, k_scale=None, v_scale=None,
                fmt: str | None = None, interleaved: bool = False, magnitude: float = 1.0,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """One layer's rotation and append in one launch: returns rope(q), and the
    pools get what append (fp32 and bf16 pools) or append_q (fmt 'int8' or 'fp8',
    with the scale pools) of rope(k_new) and v_new writes.  Shapes as append's and
    rope's; out may be q."""
    f32 = torch.float32
    dev = q.get_device()
    qs, ns, vs_ = q.stride(), k_new.stride(), v_new.stride()
    if not (dev >= 0 and q.dtype is f32 and k_new.dtype is f32 and v_new.dtype is f32 and
            positions.dtype is torch.int32 and inv_freq.dtype is torch.float64 and
            slot_mapping.dtype is torch.int64 and qs[-1] == 1 and ns[-1] == 1 and
            vs_[-1] == 1 and positions.is_contiguous() and inv_freq.is_contiguous() and
            slot_mapping.is_contiguous() and k_pool.is_contiguous() and
            v_pool.is_contiguous() and
            dev == k_new.get_device() == v_new.get_device() == positions.get_device() ==
            inv_freq.get_device() == k_pool.get_device() == v_pool.get_device() ==
            slot_mapping.get_device()):
        _rows(q, "q"), _rows(k_new, "k_new"), _rows(v_new, "v_new")  # says which and why
        _rope_tensors(positions, inv_freq)
        _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool")
        _dev(slot_mapping, "slot_mapping", torch.int64)
        _one_device(dev, ((k_new, "k_new"), (v_new, "v_new"), (positions, "positions"),
                          (inv_freq, "inv_freq"), (k_pool, "k_pool"), (v_pool, "v_pool"),
                          (slot_mapping, "slot_mapping")))
    shape, qshape, nshape = k_pool.shape, q.shape, k_new.shape
    if len(shape) != 4 or shape != v_pool.shape or k_pool.dtype is not v_pool.dtype:
        raise ValueError("k_pool and v_pool must be one layer's pools of one shape and type")
    nb, hkv, bs, d = shape
    t, hq, dq = qshape
    if nshape != (t, hkv, d) or v_new.shape != nshape or dq != d:
        raise ValueError(f"q {tuple(qshape)}, k_new {tuple(nshape)}, v_new "
                         f"{tuple(v_new.shape)} do not match pool {tuple(shape)}")
    if ns != vs_ and (t > 1 and ns[0] != vs_[0] or hkv > 1 and ns[1] != vs_[1]):
        raise ValueError("k_new and v_new must have the same strides")
    (half,) = inv_freq.shape
    if positions.shape != (t,) or slot_mapping.shape != (t,) or 2 * half > d:
        raise ValueError("positions and slot_mapping must be [n_tokens], inv_freq "
                         "[rotary_dim / 2] with rotary_dim <= head_dim")
    if fmt is None:
        code, ks, vs = _dtype_code(k_pool), None, None
    else:
        code = _qcode(fmt)
        _dev(k_pool, "k_pool", torch.uint8)
        if k_scale is None or v_scale is None:
            raise ValueError("1-byte pools need their scale pools")
        _scale_pools(k_pool, v_pool, k_scale, v_scale, code)
        _one_device(dev, ((k_scale, "k_scale"), (v_scale, "v_scale")))
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
    if out is None:
        out = q.new_empty(qshape)  # 0.8 us less than torch.empty
        os = out.stride()
    else:
        os = out.stride()
        if out.shape != qshape or out.dtype is not f32 or os[-1] != 1 or out.get_device() != dev:
            raise ValueError("out must be fp32 of q's shape with contiguous rows, on its device")
    _launch(dev, lib().rkv_rope_append, out.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), ks,
            vs, q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), os[0], os[1], qs[0], qs[1],
            ns[0], ns[1], positions.data_ptr(), inv_freq.data_ptr(), slot_mapping.data_ptr(), t,
            hq, hkv, d, 2 * half, int(interleaved), magnitude, bs, nb, code)
    return out


# ---- eviction by accumulated attention weight ------------------------------------

@functools.lru_cache(maxsize=4096)
def weights_workspace_bytes(num_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                            max_context: int) -> int:
    return int(lib().rkv_decode_weights_workspace_bytes(num_seqs, num_q_heads, num_kv_heads,
                                                        head_dim, max_context))


def _pool_code(k_pool, v_pool, k_scale, v_scale, fmt):
    """(dtype code, k_scale pointer, v_scale pointer) of pools of any format."""
    if k_pool.shape != v_pool.shape or k_pool.dtype != v_pool.dtype:
        raise ValueError("k_pool and v_pool must have one shape and type")
    if fmt is None:
        return _dtype_code(k_pool), None, None
    code = _anycode(fmt)
    _dev(k_pool, "k_pool", torch.uint8)
    if k_scale is None or v_scale is None:
        raise ValueError("1-byte pools need their scale pools")
    _scale_pools(k_pool, v_pool, k_scale, v_scale, code)
    return code, k_scale.data_ptr(), v_scale.data_ptr()


def decode_attention_weights(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                             weights: torch.Tensor, block_tables: torch.Tensor,
                             ctx_lens: torch.Tensor, scale: float | None = None, *,
                             k_scale=None, v_scale=None, fmt: str | None = None,
                             max_context: int | None = None, out: torch.Tensor | None = None,
                             workspace: torch.Tensor | None = None) -> torch.Tensor:
    """decode_attention that also adds to weights (fp32 [num_blocks, Hkv, 16])
    the softmax weight each cached row received, summed over its KV head's query
    heads.  fmt None: fp32 or bf16 pools; else a 1-byte format with its scale
    pools.  workspace: weights_workspace_bytes."""
    f32, i32 = torch.float32, torch.int32
    dev = q.get_device()
    if not (dev >= 0 and q.dtype is f32 and weights.dtype is f32 and block_tables.dtype is i32 and
            ctx_lens.dtype is i32 and q.is_contiguous() and weights.is_contiguous() and
            k_pool.is_contiguous() and v_pool.is_contiguous() and
            block_tables.is_contiguous() and ctx_lens.is_contiguous() and
            dev == k_pool.get_device() == v_pool.get_device() == weights.get_device() ==
            block_tables.get_device() == ctx_lens.get_device()):
        _dev(q, "q", f32), _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool")  # says which and why
        _dev(block_tables, "block_tables", i32), _dev(ctx_lens, "ctx_lens", i32)
        _dev(weights, "weights", f32)
        _one_device(dev, ((k_pool, "k_pool"), (v_pool, "v_pool"), (weights, "weights"),
                          (block_tables, "block_tables"), (ctx_lens, "ctx_lens")))
    shape, tables = k_pool.shape, block_tables.shape
    check_attention_shapes(q.shape, shape, tables, ctx_lens.shape)
    if weights.shape != shape[:3]:
        raise ValueError("weights must be the pools' shape without head_dim")
    code, ks, vs = _pool_code(k_pool, v_pool, k_scale, v_scale, fmt)
    if ks is not None:
        _one_device(dev, ((k_scale, "k_scale"), (v_scale, "v_scale")))
    nb, hkv, bs, d = shape
    B, hq, _ = q.shape
    mbs = tables[1]
    if max_context is None:
        max_context = mbs * bs
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.empty_like(q)
    else:
        _out_like(out, q)
    if workspace is None:  # the library checks the size of a caller's
        need = weights_workspace_bytes(B, hq, hkv, d, max_context)
        workspace = q.new_empty(max(need, 16), dtype=torch.uint8)
    else:
        _one_device(dev, ((_dev(workspace, "workspace"), "workspace"),))
    _launch(dev, lib().rkv_decode_attention_weights, out.data_ptr(), weights.data_ptr(),
            q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), ks, vs, block_tables.data_ptr(),
            mbs, ctx_lens.data_ptr(), B, hq, hkv, d, bs, nb, max_context, float(scale), code,
            workspace.data_ptr(), workspace.numel() * workspace.element_size())
    return out


def evict_select(weights: torch.Tensor, block_tables: torch.Tensor, ctx_lens: torch.Tensor,
                 budget: int, *, sinks: int = 4, recent: int = 0, max_context: int | None = None,
                 keep: torch.Tensor | None = None, new_lens: torch.Tensor | None = None):
    """The positions each KV head keeps of every sequence: its first `sinks`, its
    last `recent` and of the others the largest weights (ties to the lower
    position), `budget` in all.  weights [num_blocks, Hkv, 16] or [n_layers, ..].
    Returns (keep int32 [.., B, Hkv, budget], ascending, -1 behind the last;
    new_lens int32 [B])."""
    i32 = torch.int32
    dev = weights.get_device()
    if not (dev >= 0 and weights.dtype is torch.float32 and block_tables.dtype is i32 and
            ctx_lens.dtype is i32 and weights.is_contiguous() and block_tables.is_contiguous() and
            ctx_lens.is_contiguous() and
            dev == block_tables.get_device() == ctx_lens.get_device()):
        _dev(weights, "weights", torch.float32)  # says which and why
        _dev(block_tables, "block_tables", i32), _dev(ctx_lens, "ctx_lens", i32)
        _one_device(dev, ((block_tables, "block_tables"), (ctx_lens, "ctx_lens")))
    if weights.dim() not in (3, 4) or block_tables.dim() != 2 or ctx_lens.dim() != 1 or \
            block_tables.shape[0] != ctx_lens.shape[0]:
        raise ValueError("weights [.., num_blocks, Hkv, 16], one table row and length a sequence")
    _one_device(dev, ((keep, "keep"), (new_lens, "new_lens")))
    n_layers = weights.shape[0] if weights.dim() == 4 else 1
    nb, hkv, bs = weights.shape[-3:]
    B, mbs = block_tables.shape
    shape = (*weights.shape[:-3], B, hkv, budget)
    if keep is None:
        keep = weights.new_empty(shape, dtype=torch.int32)
    elif _dev(keep, "keep", torch.int32).shape != shape:
        raise ValueError(f"keep must be {shape}")
    if new_lens is None:
        new_lens = weights.new_empty(B, dtype=torch.int32)
    elif _dev(new_lens, "new_lens", torch.int32).shape != (B,):
        raise ValueError("new_lens must be [B]")
    _launch(dev, lib().rkv_evict_select, keep.data_ptr(), new_lens.data_ptr(),
            weights.data_ptr(), nb * hkv * bs, block_tables.data_ptr(), mbs, ctx_lens.data_ptr(),
            B, n_layers, hkv, bs, nb, budget, sinks, recent,
            mbs * bs if max_context is None else max_context)
    return keep, new_lens


def evict_compact(k_pool: torch.Tensor, v_pool: torch.Tensor, keep: torch.Tensor,
                  new_lens: torch.Tensor, src_tables: torch.Tensor, dst_tables: torch.Tensor, *,
                  k_scale=None, v_scale=None, weights: torch.Tensor | None = None,
                  fmt: str | None = None) -> None:
    """Moves the kept rows (evict_select) of every sequence and layer to positions
    0 .. new_lens[b]-1 of dst_tables (int32 [B, blocks]), with their scales and
    sums.  No destination block may be a source of the call or stand twice; the
    source blocks stay as they are for the caller to free."""
    i32 = torch.int32
    dev = k_pool.get_device()
    if not (dev >= 0 and keep.dtype is i32 and new_lens.dtype is i32 and src_tables.dtype is i32 and
            dst_tables.dtype is i32 and k_pool.is_contiguous() and v_pool.is_contiguous() and
            keep.is_contiguous() and new_lens.is_contiguous() and src_tables.is_contiguous() and
            dst_tables.is_contiguous() and
            dev == v_pool.get_device() == keep.get_device() == new_lens.get_device() ==
            src_tables.get_device() == dst_tables.get_device()):
        _dev(k_pool, "k_pool"), _dev(v_pool, "v_pool"), _dev(keep, "keep", i32)  # says which
        _dev(new_lens, "new_lens", i32), _dev(src_tables, "src_tables", i32)     # and why
        _dev(dst_tables, "dst_tables", i32)
        _one_device(dev, ((v_pool, "v_pool"), (keep, "keep"), (new_lens, "new_lens"),
                          (src_tables, "src_tables"), (dst_tables, "dst_tables")))
    if k_pool.dim() not in (4, 5):
        raise ValueError("pools must be [num_blocks, Hkv, 16, D] or [n_layers, ..]")
    code, ks, vs = _pool_code(k_pool, v_pool, k_scale, v_scale, fmt)
    if ks is not None or weights is not None:
        _one_device(dev, ((k_scale, "k_scale"), (v_scale, "v_scale"), (weights, "weights")))
    nb, hkv, bs, d = k_pool.shape[-4:]
    n_layers = k_pool.shape[0] if k_pool.dim() == 5 else 1
    B = new_lens.shape[0]
    if keep.dim() != k_pool.dim() - 1 or keep.shape[:-1] != (*k_pool.shape[:-4], B, hkv):
        raise ValueError(f"keep shape {tuple(keep.shape)} does not match pool {tuple(k_pool.shape)}")
    if src_tables.dim() != 2 or dst_tables.dim() != 2 or src_tables.shape[0] != B or \
            dst_tables.shape[0] != B:
        raise ValueError("one source and one destination table row per sequence")
    if weights is not None and _dev(weights, "weights", torch.float32).shape != k_pool.shape[:-1]:
        raise ValueError("weights must be the pools' shape without head_dim")
    _launch(dev, lib().rkv_evict_compact, k_pool.data_ptr(), v_pool.data_ptr(), ks,
            vs, weights.data_ptr() if weights is not None else None, nb * hkv * bs * d,
            nb * hkv * bs, keep.data_ptr(), new_lens.data_ptr(), keep.shape[-1],
            src_tables.data_ptr(), src_tables.shape[1], dst_tables.data_ptr(), dst_tables.shape[1],
            B, n_layers, hkv, d, bs, nb, code)


class DeviceBlockManager:
    """The FIFO paged block manager with its state in device memory
    (``rkv_dbm_*``): same ids in the same tables as the host ``PagedCache``
    for the same calls, but every operation is enqueued on the stream, so a
    decode step (reserve, slot mapping, append, attention) needs no host
    round trip.  Sequences are addressed by slot (0 .. max_seqs-1)."""

    def __init__(self, num_blocks: int, block_size: int = 16, max_seqs: int = 256,
                 max_blocks_per_seq: int = 256, device=None):
        self.device = torch.device(device if device is not None else "cuda")
        self.num_blocks, self.block_size = num_blocks, block_size
        self.max_seqs, self.max_blocks = max_seqs, max_blocks_per_seq
        s = torch.cuda.current_stream(self.device).cuda_stream
        self._h = lib().rkv_dbm_create(num_blocks, block_size, max_seqs, max_blocks_per_seq, s)
        if not self._h:
            raise _lib.RkvError(-1, lib().rkv_last_error().decode())

    def close(self) -> None:
        """Frees the device state (hipFree waits for the work in flight)."""
        if getattr(self, "_h", None):
            lib().rkv_dbm_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # interpreter shutdown
            pass

    def _s(self) -> int:
        return torch.cuda.current_stream(self.device).cuda_stream

    def _i32(self, x) -> torch.Tensor:
        return torch.as_tensor(x, dtype=torch.int32, device=self.device).contiguous()

    def reserve(self, slots, num_tokens) -> None:
        """Grow each slot's table to ceil(num_tokens / block_size) blocks
        (all or nothing; failures show in ``status()``)."""
        sl, nt = self._i32(slots), self._i32(num_tokens)
        assert sl.numel() == nt.numel()
        check(lib().rkv_dbm_reserve(self._h, sl.data_ptr(), nt.data_ptr(), sl.numel(), self._s()))

    def free(self, slots) -> None:
        sl = self._i32(slots)
        check(lib().rkv_dbm_free(self._h, sl.data_ptr(), sl.numel(), self._s()))

    def slot_mapping(self, slots, positions) -> torch.Tensor:
        sl, pos = self._i32(slots), self._i32(positions)
        out = torch.empty(sl.numel(), dtype=torch.int64, device=self.device)
        check(lib().rkv_dbm_slot_mapping(self._h, sl.data_ptr(), pos.data_ptr(), sl.numel(),
                                         out.data_ptr(), self._s()))
        return out

    def batch_tables(self, slots, max_blocks: int) -> torch.Tensor:
        sl = self._i32(slots)
        out = torch.empty((sl.numel(), max_blocks), dtype=torch.int32, device=self.device)
        check(lib().rkv_dbm_batch_tables(self._h, sl.data_ptr(), sl.numel(), out.data_ptr(),
                                         max_blocks, self._s()))
        return out

    def status(self, clear: bool = False):
        """(free blocks, error bits); synchronises the stream."""
        import ctypes as C
        nf, err = C.c_int64(0), C.c_int32(0)
        check(lib().rkv_dbm_status(self._h, C.addressof(nf), C.addressof(err), int(clear),
                                   self._s()))
        return nf.value, err.value

    def download(self):
        """(tables [max_seqs, max_blocks], lengths [max_seqs], free list front
        first) as numpy arrays; synchronises the stream."""
        import ctypes as C
        import numpy as np
        tables = np.empty((self.max_seqs, self.max_blocks), np.int32)
        lengths = np.empty(self.max_seqs, np.int32)
        free = np.empty(self.num_blocks, np.int32)
        nf = C.c_int64(0)
        check(lib().rkv_dbm_download(self._h, tables.ctypes.data, lengths.ctypes.data,
                                     free.ctypes.data, C.addressof(nf), self._s()))
        return tables, lengths, free[:nf.value].copy()


__all__ = ["append", "gather", "copy_blocks", "decode_attention", "prefill_attention",
           "append_q", "gather_q", "decode_attention_q", "workspace_bytes",
           "DeviceBlockManager", "_lib", "partition_size_for", "decode_attention_append",
           "decode_attention_append_q", "append_block_q", "prefill_attention_q",
           "rope_frequencies", "rope", "rope_append", "weights_workspace_bytes",
           "decode_attention_weights", "evict_select", "evict_compact"]
