"""4-bit latent cache and 4-bit weights of the S6 path on B200.

The bf16 ops of ``s6_ops`` / ``s6_layer`` / ``cache_export`` in their 4-bit form: rows of 17/16 bytes per latent
column instead of 4 (544 bytes for a 512-wide latent, bf16 2048), weights of 17/32 bytes per value.

* ``new_cache``          an empty 4-bit cache ``[num_blocks, 1, page, 17 * width / 16]`` (uint8)
* ``commit_rows``        rotate, quantise and scatter the rows of a step (``hla_s6_commit_rows``'s 4-bit form;
                         s6_layer.py:135-147 + unified_kv_cache_update, ouro_latent.py:127-129)
* ``history_attention``  the paged reader (s6_ops.py:117-161); ``s6_ops.history_attention`` calls it for a uint8
                         cache, ``s6_layer.attend`` and ``ouro_attention`` take such caches too
* ``gather_rows`` / ``gather_slots``  rows back as bf16 (the export's gather, cache_export.py:160-174)
* ``quantize_weight`` / ``linear``    packed weights, and ``x . w^T`` with them (register.py:45-61,
                         ouro_latent.py:109-110, 130); ``Weight`` holds one for ``ouro_attention`` and
                         ``LatentLayer.pack_writers``

Format: a group of 32 consecutive columns shares one e4m3 scale ``s``; a value is ``(n - 8) * s * ts`` with a
code ``n`` in 1..15 and one tensor scale ``ts``: ``s = e4m3(amax / (7 ts))``, ``n = 8 + rint(x / (s ts))``.  An
infinity takes the largest code of its group; a group that holds a NaN reads back as NaN throughout.  The byte layout is in include/hla_s6.h.  The tensor scales (``k_scale`` / ``v_scale`` of a cache, ``scale`` of a
weight) are not stored with the codes: every call on the same data passes the same values.  A scale covers groups
with amax between 0.11 ts and 3136 ts at full precision; ``tensor_scale`` picks one.

As everywhere in this package the ops run on CUDA tensors only, on the current stream of their device, never
synchronise and can be captured in CUDA graphs.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _lib

GROUP = 32
WEIGHT_TILE_BYTES = 1088   # HLA_S6_Q4_WEIGHT_TILE_BYTES
LINEAR_TOKENS = 65535 * 256   # the most tokens of one linear (a grid of tiles of 256)
BF16, U8, I32, I64 = torch.bfloat16, torch.uint8, torch.int32, torch.int64


def row_bytes(width):
    """Bytes of one 4-bit cache row (K and V) of latent width ``width``."""
    return 17 * width // 16


def cache_width(cache):
    """Latent width of a 4-bit cache."""
    return cache.shape[-1] * 16 // 17


def tensor_scale(amax):
    """The smallest power of two that lets the largest group scale reach e4m3's range for values up to ``amax``
    (a float), from 2^-126 on; a power of two keeps every stored value exact in bf16."""
    if not math.isfinite(amax):
        raise ValueError(f'the largest value must be finite (got {amax})')
    return 2.0 ** math.ceil(math.log2(max(amax / (7 * 448), 2.0 ** -126))) if amax > 0 else 1.0


def new_cache(num_blocks, page, width, device='cuda'):
    """A zeroed 4-bit latent cache (every row reads as zeros)."""
    if width not in (256, 512, 1024) or page < 16 or page % 16:
        raise ValueError('a 4-bit latent cache has width 256, 512 or 1024 and a page of a multiple of 16 rows')
    return torch.zeros(num_blocks, 1, page, row_bytes(width), dtype=U8, device=device)


_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _device_of(first, *rest):
    """The index of the one CUDA device that every tensor is on."""
    index = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != index:
            index = -1
    if index < 0:
        raise ValueError('S6 4-bit ops take CUDA tensors of one device (no CPU path exists)')
    return index


_entries = {}   # the library's functions by name, looked up once


def _launch(index, name, *args):
    """Entry point ``name`` with ``args`` and the current stream of device ``index``, which is made current for the
    launch.  (Plain ints and the raw stream handle, and outputs by the quickest of torch's constructors: the calls of
    one token's step cost more on the host than on the device.)"""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


def _address(t):
    return None if t is None else t.data_ptr()


def _check_flag(error_flag):
    if error_flag is not None and (error_flag.dtype is not I32 or error_flag.numel() < 1):
        raise ValueError('error_flag must be int32 [1]')


def _cache_geometry(cache, width):
    """``(num_blocks, block stride in bytes, page)`` of a 4-bit cache of latent width ``width``."""
    shape, bytes_ = cache.shape, 17 * width // 16
    if len(shape) != 4 or shape[1] != 1 or shape[3] != bytes_ or cache.dtype is not U8:
        raise ValueError(f'a 4-bit latent cache of width {width} must be uint8 [num_blocks, 1, page, {bytes_}], got '
                         f'{cache.dtype} {tuple(shape)}')
    stride = cache.stride()
    if stride[3] != 1 or stride[2] != bytes_:
        raise ValueError('the bytes of a 4-bit cache page must be contiguous')
    return shape[0], stride[0], shape[2]


def _block_table(table):
    """``(row stride, rows, columns)`` of a block table."""
    shape, stride = table.shape, table.stride()
    if table.dtype is not I32 or len(shape) != 2 or stride[1] != 1:
        raise ValueError('block_table must be int32 [rows, max_blocks] with a unit last-dim stride')
    return stride[0], shape[0], shape[1]


def history_attention(q_lat, cache, block_table, ctx, scale, num_kv_splits, workspace, k_scale=1.0, v_scale=1.0,
                      empty=None, error_flag=None):
    """``s6_ops.history_attention`` over a 4-bit cache: ``(o [T, H, W] bf16, lse [H, T] fp32)`` of the softmax of
    ``q_lat [T, H, W]`` over the first ``ctx[t]`` rows; empty rows give ``o = 0``, ``lse = -inf``.
    A NaN in a query or in a key makes the rows that meet it NaN, ``lse`` too.
    ``error_flag`` (int32 [1], optional) receives 5 for a block-table entry outside the cache."""
    stride = q_lat.stride()
    if len(stride) != 3 or q_lat.dtype is not BF16 or stride[2] != 1:
        raise ValueError('q_lat must be bf16 [T, H, W] with a unit last-dim stride')
    T, H, W = q_lat.shape
    nb, sb, page = _cache_geometry(cache, W)
    bt_stride, bt_rows, bt_cols = _block_table(block_table)
    if ctx.dtype is not I32 or ctx.shape != (T,) or bt_rows < T:
        raise ValueError('ctx must be int32 [T] and block_table hold a row per token')
    if empty is not None:
        if empty.shape != (T,):
            raise ValueError('empty must be [T]')
        empty = empty.contiguous() if empty.dtype in (torch.bool, torch.uint8) else (empty != 0)
    _check_flag(error_flag)
    index = _device_of(q_lat, cache, block_table, ctx, empty, error_flag)
    buffer = workspace.ensure(q_lat.device)   # (after the check: a workspace keeps the device of its first use)
    _device_of(q_lat, buffer)
    need = T * H * num_kv_splits * (W + 1)
    if need > buffer.numel():
        raise RuntimeError(f'S6 workspace overflow: need {need} floats, have {buffer.numel()}')
    o = q_lat.new_empty(T, H, W)
    lse = buffer.new_empty(H, T)
    ctx = ctx.contiguous()
    _launch(index, 'hla_s6_history_attention_q4', q_lat.data_ptr(), stride[0], stride[1], cache.data_ptr(), nb, sb,
            block_table.data_ptr(), bt_stride, bt_cols, ctx.data_ptr(), _address(empty), T, H, W, page, float(scale),
            int(num_kv_splits), buffer.data_ptr(), need, float(k_scale), float(v_scale), o.data_ptr(), H * W, W,
            lse.data_ptr(), _address(error_flag))
    return o, lse


def commit_rows(row, positions, table, cache, block_table, query_start_loc, k_scale=1.0, v_scale=1.0):
    """Commit ``row [T, 2 W]`` (K | V, bf16): the K half latent-RoPE'd by ``table [max_position, W]`` at
    ``positions [T]`` (int64), both halves quantised and stored at ``block_table[request, pos // page] * page +
    pos % page``.  Returns the slots (int64 [T]); padding tokens (``t >= query_start_loc[-1]``) and positions
    without a block in the cache are skipped, their slot is -1.  Two tokens of one call must not share a slot."""
    stride = row.stride()
    if len(stride) != 2 or row.dtype is not BF16 or stride[1] != 1 or row.shape[1] & 1:
        raise ValueError('row must be bf16 [T, 2 * width] with a unit last-dim stride')
    T, W = row.shape
    W //= 2
    nb, sb, page = _cache_geometry(cache, W)
    tab_rows, tab_stride = table.shape, table.stride()
    if len(tab_stride) != 2 or table.dtype is not BF16 or tab_stride[1] != 1 or tab_rows[1] != W:
        raise ValueError(f'table must be bf16 [max_position, {W}] = [cos | sin]')
    bt_stride, bt_rows, bt_cols = _block_table(block_table)
    requests = query_start_loc.numel() - 1
    if (positions.dtype is not I64 or positions.shape != (T,) or query_start_loc.dtype is not I32
            or query_start_loc.dim() != 1 or bt_rows < requests):
        raise ValueError('positions must be int64 [T], query_start_loc int32 [R + 1], block_table [R, max_blocks]')
    index = _device_of(row, positions, table, cache, block_table, query_start_loc)
    positions, query_start_loc = positions.contiguous(), query_start_loc.contiguous()
    slots = positions.new_empty(T)
    _launch(index, 'hla_s6_commit_rows_q4', row.data_ptr(), stride[0], W, positions.data_ptr(), table.data_ptr(),
            tab_stride[0], tab_rows[0], cache.data_ptr(), nb, sb, page, block_table.data_ptr(),
            bt_stride, bt_cols, query_start_loc.data_ptr(), requests, T, float(k_scale),
            float(v_scale), slots.data_ptr())
    return slots


def _gather(cache, blocks, slots, rows, k_scale, v_scale, out, error_flag):
    W = cache.shape[-1] * 16 // 17
    nb, sb, page = _cache_geometry(cache, W)
    index = blocks if slots is None else slots
    if index.dim() != 1 or index.dtype is not (I32 if slots is None else I64):
        raise ValueError('blocks must be int32 [n], slots int64 [n]')
    if rows < 0 or (slots is None and -(-rows // page) > blocks.shape[0]):
        raise IndexError('the block list does not cover the rows')
    if out is not None and (out.shape != (rows, 2 * W) or out.dtype is not BF16 or out.stride(-1) != 1):
        raise ValueError(f'out must be bf16 [{rows}, {2 * W}] with a unit last-dim stride')
    _check_flag(error_flag)
    device = _device_of(cache, index, out, error_flag)
    index = index.contiguous()
    if out is None:
        out = torch.empty_strided((rows, 2 * W), (2 * W, 1), dtype=BF16, device=cache.device)
    if rows:
        at = index.data_ptr()
        _launch(device, 'hla_s6_gather_rows_q4', cache.data_ptr(), nb, sb, W, page, at if slots is None else None,
                None if slots is None else at, rows, float(k_scale), float(v_scale), out.data_ptr(),
                out.stride(0), _address(error_flag))
    return out


def gather_rows(cache, blocks, length, k_scale=1.0, v_scale=1.0, out=None, error_flag=None):
    """Rows 0 .. length - 1 of a request as bf16 ``[length, 2 W]`` (rotated K | V): row i is row ``i % page`` of
    block ``blocks[i // page]`` (int32).  A block outside the cache gives zeros and sets ``error_flag`` to 5."""
    return _gather(cache, blocks, None, int(length), k_scale, v_scale, out, error_flag)


def gather_slots(cache, slots, k_scale=1.0, v_scale=1.0, out=None, error_flag=None):
    """The rows at ``slots`` (int64, as ``commit_rows`` returns them; -1 gives zeros) as bf16 ``[n, 2 W]``."""
    return _gather(cache, None, slots, slots.shape[0], k_scale, v_scale, out, error_flag)


def weight_tiles(out_features, in_features):
    """Shape of a packed weight: ``[ceil(out / 16), ceil(in / 128), 1088]`` (uint8)."""
    return -(-out_features // 16), -(-in_features // 128), WEIGHT_TILE_BYTES


def quantize_weight(weight, scale=None):
    """``(packed, scale)`` of a bf16 weight ``[N, K]``, K a multiple of 32.  ``scale`` defaults to
    ``tensor_scale`` of its largest value (which reads it back: call this once, at load time; a weight with values
    that are not finite is then refused)."""
    if weight.dim() != 2 or weight.dtype is not BF16 or weight.stride(-1) != 1:
        raise ValueError('weight must be bf16 [N, K] with a unit last-dim stride')
    N, K = weight.shape
    if K < GROUP or K % GROUP or N < 1:
        raise ValueError('a 4-bit weight needs in_features a multiple of 32')
    index = _device_of(weight)
    if scale is None:
        amax = float(weight.abs().amax())
        if not math.isfinite(amax):
            raise ValueError('the weight holds values that are not finite')
        scale = tensor_scale(amax)
    packed = weight.new_empty(weight_tiles(N, K), dtype=U8)
    _launch(index, 'hla_s6_quantize_weight_q4', weight.data_ptr(), weight.stride(0), N, K, scale, packed.data_ptr())
    return packed, float(scale)


def _check_rows(y, T, N):
    if y.shape != (T, N) or y.dtype is not BF16 or y.stride(1) != 1:
        raise ValueError(f'residual and out must be bf16 [{T}, {N}] with a unit last-dim stride')


def linear(x, packed, out_features, scale, residual=None, out=None, error_flag=None):
    """``bf16(scale * x . w^T + residual)`` for ``x [T, K]`` bf16 and the packed weight ``[N, K]``: fp32 sums, one
    rounding.  ``residual`` and ``out`` are bf16 ``[T, N]``; ``out`` may be ``residual``, and overlaps no other input.
    Rows of x start at 16-byte boundaries.  ``error_flag`` (int32 [1], optional) receives 1 or 2 where a kernel's wait
    ran out, whose output is then wrong."""
    stride = x.stride()
    if len(stride) != 2 or x.dtype is not BF16 or stride[1] != 1:
        raise ValueError('x must be bf16 [T, K] with a unit last-dim stride')
    T, K = x.shape
    if T > LINEAR_TOKENS:
        raise ValueError(f'a 4-bit linear takes at most {LINEAR_TOKENS} tokens, got {T}')
    N = out_features
    if (packed.dtype is not U8 or packed.shape != (-(-N // 16), -(-K // 128), WEIGHT_TILE_BYTES)
            or not packed.is_contiguous()):
        raise ValueError(f'packed must be contiguous uint8 {list(weight_tiles(N, K))}, got {packed.dtype} '
                         f'{list(packed.shape)}')
    x_stride = stride[0] if T > 1 else K
    if x_stride < K:   # rows that overlap (an expanded x)
        x, x_stride = x.contiguous(), K
    if residual is not None:
        _check_rows(residual, T, N)
    if out is not None:
        _check_rows(out, T, N)
    _check_flag(error_flag)
    index = _device_of(x, packed, residual, out, error_flag)
    fresh = out is None
    if fresh:
        out = x.new_empty(T, N)
    _launch(index, 'hla_s6_linear_q4_checked', x.data_ptr(), x_stride, packed.data_ptr(), T, N, K, float(scale),
            _address(residual), 0 if residual is None else residual.stride(0), out.data_ptr(),
            N if fresh else out.stride(0), _address(error_flag))
    return out


@dataclass(frozen=True)
class Weight:
    """A packed weight with what its calls need: the weights of ``ouro_attention.LatentAttention`` and of
    ``latent.LatentLayer``'s writers may be of this kind."""
    packed: torch.Tensor
    out_features: int
    scale: float

    @classmethod
    def of(cls, weight, scale=None):
        """The 4-bit copy of a bf16 weight ``[N, K]`` (``quantize_weight``)."""
        packed, scale = quantize_weight(weight, scale)
        return cls(packed, weight.shape[0], scale)

    def linear(self, x, residual=None, out=None, error_flag=None):
        return linear(x, self.packed, self.out_features, self.scale, residual, out, error_flag)
