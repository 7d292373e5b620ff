"""An 8-bit paged KV cache: its write, the attention that reads it, and the layout of a batch.

Keys and values are held in tiles of 16 tokens of one KV head as e4m3 codes with one power-of-two
scale a tile (``include/cdb_amd.h``, "8-bit KV cache"): half the bytes of a bf16 cache, and three fifths
of the time of a decode step's attention (256 rows, 16 heads x 128: 107-110 us a layer against 178). The calls
mirror those of the pool in the model's type (``ops``): ``write`` beside ``rope_kv_write``, ``decode_attention``
beside ``paged_decode_attention``, ``prefill_attention`` beside ``prefill_attention``; ``batch_layout`` builds
on the GPU what they take as block tables, slots and attention tiles.

Each ``*_raw`` function checks its arguments on the host and makes one C call on torch's current stream
without allocating, so it can be captured into a HIP graph; the ``torch.ops.cdb.kv8_*`` ops wrap them.
Tensors must lie on the current device.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from .ops import _ptr, _stream, dtype_code

TILE = 16  # tokens of a cache tile
_E4M3, _U8, _I32, _I64 = torch.float8_e4m3fn, torch.uint8, torch.int32, torch.int64
PREFILL_TILE = 128  # query tokens of an attention tile

LAYOUT_TOKENS_FULL = _lib.CDB_LAYOUT_TOKENS_FULL
LAYOUT_TILES_FULL = _lib.CDB_LAYOUT_TILES_FULL
LAYOUT_NO_BLOCKS = _lib.CDB_LAYOUT_NO_BLOCKS
LAYOUT_BAD_REQUEST = _lib.CDB_LAYOUT_BAD_REQUEST


@dataclass(frozen=True)
class Kv8Pool:
    """The cache: ``codes`` float8_e4m3fn ``[layers, 2, blocks, Hkv, block_size / 16, 16 * D]`` and
    ``scales`` uint8 ``[layers, 2, blocks, Hkv, block_size / 16]`` (b, from 1 to 254, stands for
    2 ** (b - 127); 0 is read as 1 and 255 as 254), keys at index 0 of dim 1 and values at 1."""

    codes: torch.Tensor
    scales: torch.Tensor

    def __post_init__(self) -> None:
        self._check()

    def _check(self) -> tuple[torch.Size, torch.Size, tuple[int, int, int, int, int]]:
        c, s = self.codes, self.scales
        if c.dtype is not torch.float8_e4m3fn or s.dtype is not torch.uint8:
            raise TypeError("an 8-bit pool holds float8_e4m3fn codes and uint8 scales")
        shape = c.shape
        if len(shape) != 6 or shape[1] != 2 or s.shape != shape[:5] or shape[5] % TILE:
            raise ValueError("codes must be [layers, 2, blocks, Hkv, block_size / 16, 16 * D] and scales match them")
        if not c.is_contiguous() or not s.is_contiguous() or c.device != s.device:
            raise ValueError("codes and scales must be contiguous and on one device")
        layers, _, blocks, heads, tiles, tile = shape
        facts = (shape, s.shape, (layers, blocks, heads, tile // TILE, tiles * TILE))
        object.__setattr__(self, "_facts", facts)
        return facts

    def _resolve(self) -> tuple[int, int, tuple[int, int, int, int, int]]:
        """(codes, scales, (layers, blocks, Hkv, D, block_size)) of the tensors as they are now. Every call asks: a
        pool may be a copy, or its tensors may have been given other memory."""

        c, s, facts = self.codes, self.scales, self._facts
        if c.shape != facts[0] or s.shape != facts[1] or c.dtype is not _E4M3 or s.dtype is not _U8 \
                or not c.is_contiguous() or not s.is_contiguous():
            facts = self._check()
        return c.data_ptr(), s.data_ptr(), facts[2]

    @classmethod
    def allocate(cls, num_cache_layers: int, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                 device: torch.device | str) -> "Kv8Pool":
        """A pool of zeros."""

        if block_size < TILE or block_size & (block_size - 1):
            raise ValueError(f"block_size must be a power of two of at least {TILE}, got {block_size}")
        shape = (num_cache_layers, 2, num_blocks, num_kv_heads, block_size // TILE)
        codes = torch.zeros((*shape, TILE * head_dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        return cls(codes, torch.zeros(shape, dtype=torch.uint8, device=device))

    @property
    def num_cache_layers(self) -> int:
        return self.codes.shape[0]

    @property
    def num_blocks(self) -> int:
        return self.codes.shape[2]

    @property
    def num_kv_heads(self) -> int:
        return self.codes.shape[3]

    @property
    def head_dim(self) -> int:
        return self.codes.shape[5] // TILE

    @property
    def block_size(self) -> int:
        return self.codes.shape[4] * TILE

    def dequantize(self, layer: int, blocks: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """fp32 keys and values ``[len(blocks) * block_size, Hkv, D]`` of the named blocks of a cache layer, for
        inspection and tests (torch indexing, not a kernel)."""

        d = self.head_dim
        raw = self.codes.view(torch.uint8)[layer][:, blocks].view(torch.float8_e4m3fn).float()
        scale = torch.ldexp(torch.ones((), device=raw.device, dtype=torch.float64),
                            self.scales[layer][:, blocks].int().clamp(1, 254) - 127).float()
        raw = raw * scale[..., None]
        k = raw[0].unflatten(-1, (d // 16, TILE, 16)).transpose(-3, -2).flatten(-2)   # [blocks, Hkv, tiles, 16, D]
        v = raw[1].unflatten(-1, (4, d, 4)).transpose(-2, -1).flatten(-3, -2)
        return tuple(x.permute(0, 2, 3, 1, 4).flatten(0, 2) for x in (k, v))


# A decode step's call takes about as long as its kernel, so the checks below touch each tensor property once.


def _require_here(*tensors: torch.Tensor | None) -> None:
    """Every tensor on the current device, whose stream the launch goes to."""

    devices = {t.get_device() for t in tensors if t is not None}
    if len(devices) == 1 and -1 not in devices and torch._C._cuda_getDevice() in devices:
        return
    for t in tensors:
        if t is not None and t.get_device() < 0:
            raise RuntimeError("CDB kernels run on the GPU only; got a tensor on " + str(t.device))
    here = torch._C._cuda_getDevice()
    for t in tensors:
        if t is not None and t.get_device() != here:
            raise RuntimeError(f"got a tensor on {t.device} while cuda:{here} is the current device")


def _check_ints(name: str, t: torch.Tensor, n: int) -> None:
    if t.dtype is not _I32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous with {n} entries")


def _check_table(block_table: torch.Tensor) -> tuple[int, int]:
    if block_table.dtype is not torch.int32:
        raise TypeError(f"block_table must be int32, got {block_table.dtype}")
    if block_table.dim() != 2 or not block_table.is_contiguous():
        raise ValueError("block_table must be a contiguous [rows, width]")
    return tuple(block_table.shape)


def _check_rope(rope_style: int, cos: torch.Tensor | None, sin: torch.Tensor | None, head_dim: int) -> int:
    """The tables' positions; raises on tables that do not fit."""

    if rope_style == 0:
        return 0
    if rope_style not in (1, 2):
        raise ValueError(f"rope_style must be 0, 1 or 2, got {rope_style}")
    if cos is None or sin is None or cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise ValueError("rope tables must be float32 [max_positions, D/2]")
    shape = cos.shape
    if len(shape) != 2 or shape[1] != head_dim // 2 or sin.shape != shape or not cos.is_contiguous() \
            or not sin.is_contiguous():
        raise ValueError("rope tables must be contiguous float32 [max_positions, D/2]")
    return shape[0]


def _check_bias(name: str, bias: torch.Tensor | None, heads: int, dim: int, dtype: torch.dtype) -> None:
    if bias is None:
        return
    if bias.shape != (heads, dim) or bias.dtype is not dtype or not bias.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{heads}, {dim}] tensor of q's dtype")


def _row_stride(name: str, t: torch.Tensor, rows: int, heads: int, head_dim: int) -> int:
    """Elements between rows of a [rows, heads, D] tensor whose heads are dense; a single row's is its own size."""

    row, head, element = t.stride()
    if element != 1 or (head != head_dim and heads > 1):
        raise ValueError(f"{name} must have contiguous heads and head dimension (the row stride may differ)")
    if rows <= 1:
        return heads * head_dim
    if row < heads * head_dim:
        raise ValueError(f"{name}'s rows overlap")
    return row


def write_raw(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, q_out: torch.Tensor | None, pool: Kv8Pool,
              layer: int, rows: torch.Tensor, positions: torch.Tensor, rope_cos: torch.Tensor | None,
              rope_sin: torch.Tensor | None, rope_style: int, q_bias: torch.Tensor | None,
              k_bias: torch.Tensor | None) -> None:
    """Launch ``cdb_kv8_write``: code T tokens' rotated keys and their values into slots ``rows`` of cache layer
    ``layer`` and put the rotated queries into ``q_out`` (q and q_out None: keys and values alone). q, k and v
    may be token-strided views. The tokens of one tile follow each other at consecutive slots; a negative slot
    is padding, whose q_out is left as it was. A token left out between others of its tile (padding, a slot or
    position out of range) keeps its place in the call."""

    codes, scales, (layers, blocks, heads_kv, dim, block) = pool._resolve()
    shape, dt = k.shape, k.dtype
    if len(shape) != 3 or shape[1] != heads_kv or shape[2] != dim or v.shape != shape or v.dtype is not dt:
        raise ValueError(f"k and v must be [T, {heads_kv}, {dim}] of one dtype")
    tokens = shape[0]
    heads = q_ptr = out_ptr = q_stride = 0
    if (q is None) != (q_out is None):
        raise ValueError("q and q_out come together")
    if q is not None:
        shape = q.shape
        if len(shape) != 3 or shape[0] != tokens or shape[2] != dim or q.dtype is not dt:
            raise ValueError(f"q must be [{tokens}, H, {dim}] of k's dtype")
        heads = shape[1]
        if q_out.shape != shape or q_out.dtype is not dt or not q_out.is_contiguous():
            raise ValueError("q_out must be contiguous and match q")
        q_ptr, out_ptr, q_stride = q.data_ptr(), q_out.data_ptr(), _row_stride("q", q, tokens, heads, dim)
    if rows.dtype is not torch.int64 or positions.dtype is not torch.int32:
        raise TypeError("rows must be int64 and positions int32")
    if rows.numel() < tokens or positions.numel() < tokens or not rows.is_contiguous() \
            or not positions.is_contiguous():
        raise ValueError("rows and positions must be contiguous with an entry per token")
    if not 0 <= layer < layers:
        raise ValueError("layer out of range")
    max_positions = _check_rope(rope_style, rope_cos, rope_sin, dim)
    _check_bias("q_bias", q_bias, heads, dim, dt)
    _check_bias("k_bias", k_bias, heads_kv, dim, dt)
    kv_stride = _row_stride("k", k, tokens, heads_kv, dim)
    if _row_stride("v", v, tokens, heads_kv, dim) != kv_stride:
        raise ValueError("k and v must share one token stride")
    _require_here(q, k, v, q_out, pool.codes, pool.scales, rows, positions, rope_cos, rope_sin, q_bias, k_bias)
    code = _lib.lib().cdb_kv8_write(
        q_ptr or None, k.data_ptr(), v.data_ptr(), out_ptr or None, codes, scales, layers, blocks, layer,
        rows.data_ptr(), positions.data_ptr(), _ptr(rope_cos), _ptr(rope_sin), rope_style, max_positions,
        _ptr(q_bias), _ptr(k_bias), tokens, heads, heads_kv, dim, block, q_stride, kv_stride, dtype_code(dt),
        _stream())
    if code:
        _lib.check(code, "cdb_kv8_write")


@torch.library.custom_op("cdb::kv8_write", mutates_args=("codes", "scales"), device_types="cuda")
def write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, layer: int,
          rows: torch.Tensor, positions: torch.Tensor, rope_cos: torch.Tensor | None, rope_sin: torch.Tensor | None,
          rope_style: int, q_bias: torch.Tensor | None, k_bias: torch.Tensor | None) -> torch.Tensor:
    """Rotate and append T tokens to the 8-bit cache; returns the rotated queries [T, H, D] (zeros for padding
    tokens, whose slot is negative)."""

    q_rot = q.new_zeros(q.shape)
    write_raw(q, k, v, q_rot, Kv8Pool(codes, scales), layer, rows, positions, rope_cos, rope_sin, rope_style, q_bias,
              k_bias)
    return q_rot


@write.register_fake
def _(q, k, v, codes, scales, layer, rows, positions, rope_cos, rope_sin, rope_style, q_bias, k_bias):
    return q.new_empty(q.shape)


def decode_workspace_bytes(num_rows: int, num_heads: int, num_kv_heads: int, head_dim: int, max_seqlen: int) -> int:
    """Workspace of decode launches of up to ``num_rows`` rows whose positions are below ``max_seqlen``. Rows with
    longer contexts are served too, in fewer and longer chunks, whose number (and with it the rounding of such a row)
    depends on how many rows share the workspace; with this size, a row's bits do not depend on its batch."""

    n = int(_lib.lib().cdb_kv8_decode_workspace_bytes(num_rows, num_heads, num_kv_heads, head_dim, max_seqlen))
    if n < 0:
        raise ValueError("invalid arguments for the decode workspace size")
    return n


def decode_attention_raw(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, pool: Kv8Pool,
                         cache_layer: torch.Tensor | None, cache_layer0: int, block_table: torch.Tensor,
                         table_row: torch.Tensor | None, seqlens: torch.Tensor, rope_cos: torch.Tensor | None,
                         rope_sin: torch.Tensor | None, rope_style: int, q_bias: torch.Tensor | None,
                         k_bias: torch.Tensor | None, out: torch.Tensor, workspace: torch.Tensor,
                         scale: float) -> torch.Tensor:
    """Launch ``cdb_kv8_decode_attention``: append each row's new token at position ``seqlens[b]`` and attend over
    positions 0..seqlens[b] (negative: a padding row, zero output). Arguments as ``ops.paged_decode_attention_raw``
    without its chunking; ``workspace`` is any dense tensor of ``decode_workspace_bytes`` bytes. Calls that may
    overlap need a workspace each."""

    codes, scales, (layers, blocks, heads_kv, dim, block) = pool._resolve()
    shape, dt = q.shape, q.dtype
    if len(shape) != 3 or shape[2] != dim:
        raise ValueError(f"q must be [rows, H, {dim}]")
    num_rows, num_heads = shape[0], shape[1]
    kv_shape = k_new.shape
    if kv_shape != (num_rows, heads_kv, dim) or v_new.shape != kv_shape:
        raise ValueError(f"k_new and v_new must be [{num_rows}, {heads_kv}, {dim}]")
    if k_new.dtype is not dt or v_new.dtype is not dt:
        raise TypeError("q, k_new and v_new must share a dtype")
    if num_heads == 0 or num_heads % heads_kv:
        raise ValueError(f"{num_heads} query heads cannot share {heads_kv} KV heads evenly")
    if out.shape != shape or out.dtype is not dt or not out.is_contiguous():
        raise ValueError("out must be contiguous and match q")
    table_rows, width = _check_table(block_table)
    _check_ints("seqlens", seqlens, num_rows)
    if table_row is not None:
        _check_ints("table_row", table_row, num_rows)
    elif table_rows < num_rows:
        raise ValueError("block_table needs a row per batch row when table_row is not given")
    if cache_layer is not None:
        _check_ints("cache_layer", cache_layer, num_rows)
    max_positions = _check_rope(rope_style, rope_cos, rope_sin, dim)
    _check_bias("q_bias", q_bias, num_heads, dim, dt)
    _check_bias("k_bias", k_bias, heads_kv, dim, dt)
    if not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    q_stride = _row_stride("q", q, num_rows, num_heads, dim)
    kv_stride = _row_stride("k_new", k_new, num_rows, heads_kv, dim)
    if _row_stride("v_new", v_new, num_rows, heads_kv, dim) != kv_stride:
        raise ValueError("k_new and v_new must share a row stride")
    _require_here(q, k_new, v_new, pool.codes, pool.scales, cache_layer, block_table, table_row, seqlens, rope_cos,
                  rope_sin, q_bias, k_bias, out, workspace)
    code = _lib.lib().cdb_kv8_decode_attention(
        q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), codes, scales, layers, blocks, _ptr(cache_layer),
        cache_layer0, block_table.data_ptr(), _ptr(table_row), table_rows, width, seqlens.data_ptr(),
        _ptr(rope_cos), _ptr(rope_sin), rope_style, max_positions, _ptr(q_bias), _ptr(k_bias), out.data_ptr(),
        workspace.data_ptr(), workspace.nbytes, num_rows, num_heads, heads_kv, dim, block, scale,
        q_stride, kv_stride, dtype_code(dt), _stream())
    if code:
        _lib.check(code, "cdb_kv8_decode_attention")
    return out


@torch.library.custom_op("cdb::kv8_decode_attention", mutates_args=("codes", "scales", "workspace"),
                         device_types="cuda")
def decode_attention(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, codes: torch.Tensor,
                     scales: torch.Tensor, cache_layer: torch.Tensor | None, cache_layer0: int,
                     block_table: torch.Tensor, table_row: torch.Tensor | None, seqlens: torch.Tensor,
                     rope_cos: torch.Tensor | None, rope_sin: torch.Tensor | None, rope_style: int,
                     q_bias: torch.Tensor | None, k_bias: torch.Tensor | None, workspace: torch.Tensor,
                     scale: float) -> torch.Tensor:
    """Paged decode attention over the 8-bit cache with fused rotation and append; see ``decode_attention_raw``."""

    out = q.new_empty(q.shape)
    return decode_attention_raw(q, k_new, v_new, Kv8Pool(codes, scales), cache_layer, cache_layer0, block_table,
                                table_row, seqlens, rope_cos, rope_sin, rope_style, q_bias, k_bias, out, workspace,
                                scale)


@decode_attention.register_fake
def _(q, k_new, v_new, codes, scales, cache_layer, cache_layer0, block_table, table_row, seqlens, rope_cos, rope_sin,
      rope_style, q_bias, k_bias, workspace, scale):
    return q.new_empty(q.shape)


def prefill_splits(num_tiles: int, num_heads: int, num_kv_heads: int, longest: int, num_cus: int = 256) -> int:
    """Parts that a prefill launch cuts each tile's key range into: enough to give every CU two workgroups, while
    a part keeps at least 512 keys of the longest range ``longest`` (cached and new tokens of a sequence), and at
    most 64. A sequence's rounding depends on the number of parts: pass a fixed one where that must not follow from
    the batch. Heads that share keys take a workgroup each all the same, so ``num_kv_heads`` makes no difference."""

    del num_kv_heads
    want = -(-2 * num_cus // max(1, num_tiles * num_heads))
    return max(1, min(want, longest // 512, 64))


def prefill_workspace_bytes(num_tiles: int, splits: int, num_heads: int, head_dim: int) -> int:
    n = int(_lib.lib().cdb_kv8_prefill_workspace_bytes(num_tiles, splits, num_heads, head_dim))
    if n < 0:
        raise ValueError("invalid arguments for the prefill workspace size")
    return n


def prefill_attention_raw(q: torch.Tensor, pool: Kv8Pool, layer: int, block_table: torch.Tensor,
                          table_row: torch.Tensor, cu_q: torch.Tensor, past: torch.Tensor, tile_seq: torch.Tensor,
                          tile_q0: torch.Tensor, out: torch.Tensor, scale: float, splits: int = 1,
                          workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Launch ``cdb_kv8_prefill_attention``: causal attention of rotated queries q [T, H, D] over cache layer
    ``layer``, whose keys and values hold the chunk's own tokens already. Sequences, block table and tiles as
    ``ops.prefill_attention_raw`` (``tile_seq[n] < 0``: no tile); ``splits`` from ``prefill_splits`` with a
    workspace of ``prefill_workspace_bytes`` bytes when above 1. Calls that may overlap need a workspace each."""

    codes, scales, (layers, blocks, heads_kv, dim, block) = pool._resolve()
    shape, dt = q.shape, q.dtype
    if len(shape) != 3 or shape[2] != dim or not q.is_contiguous():
        raise ValueError(f"q must be a contiguous [T, H, {dim}]")
    num_heads = shape[1]
    if out.shape != shape or out.dtype is not dt or not out.is_contiguous():
        raise ValueError("out must be contiguous and match q")
    if num_heads == 0 or num_heads % heads_kv:
        raise ValueError(f"{num_heads} query heads cannot share {heads_kv} KV heads evenly")
    num_seqs, num_tiles = past.numel(), tile_seq.numel()
    table_rows, width = _check_table(block_table)
    for name, t, n in (("past", past, num_seqs), ("cu_q", cu_q, num_seqs + 1), ("table_row", table_row, num_seqs),
                       ("tile_seq", tile_seq, num_tiles), ("tile_q0", tile_q0, num_tiles)):
        _check_ints(name, t, n)
    if not 0 <= layer < layers:
        raise ValueError("layer out of range")
    if splits > 1 and workspace is None:
        raise ValueError("split launches need a workspace")
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    _require_here(q, pool.codes, pool.scales, block_table, table_row, cu_q, past, tile_seq, tile_q0, out, workspace)
    code = _lib.lib().cdb_kv8_prefill_attention(
        q.data_ptr(), codes, scales, layers, blocks, layer, block_table.data_ptr(), table_row.data_ptr(), table_rows,
        width, cu_q.data_ptr(), past.data_ptr(), num_seqs, tile_seq.data_ptr(), tile_q0.data_ptr(), num_tiles,
        out.data_ptr(), shape[0], splits, _ptr(workspace), 0 if workspace is None else workspace.nbytes, num_heads,
        heads_kv, dim, block, scale, dtype_code(dt), _stream())
    if code:
        _lib.check(code, "cdb_kv8_prefill_attention")
    return out


@torch.library.custom_op("cdb::kv8_prefill_attention", mutates_args=("workspace",), device_types="cuda")
def prefill_attention(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, layer: int,
                      block_table: torch.Tensor, table_row: torch.Tensor, cu_q: torch.Tensor, past: torch.Tensor,
                      tile_seq: torch.Tensor, tile_q0: torch.Tensor, scale: float, splits: int,
                      workspace: torch.Tensor | None) -> torch.Tensor:
    """Varlen causal prefill attention over the 8-bit cache; see ``prefill_attention_raw``."""

    out = q.new_empty(q.shape)
    return prefill_attention_raw(q, Kv8Pool(codes, scales), layer, block_table, table_row, cu_q, past, tile_seq,
                                 tile_q0, out, scale, splits, workspace)


@prefill_attention.register_fake
def _(q, codes, scales, layer, block_table, table_row, cu_q, past, tile_seq, tile_q0, scale, splits, workspace):
    return q.new_empty(q.shape)


@dataclass(frozen=True)
class BatchLayout:
    """What ``batch_layout`` writes: ``cu_q`` [S + 1], ``positions`` int32 and ``rows`` int64 [tokens] (-1 behind
    the last token), ``tile_seq`` and ``tile_q0`` [tiles] ((-1, 0) behind the last), ``counts`` [tokens, tiles,
    blocks taken, LAYOUT_* bits]."""

    cu_q: torch.Tensor
    positions: torch.Tensor
    rows: torch.Tensor
    tile_seq: torch.Tensor
    tile_q0: torch.Tensor
    counts: torch.Tensor

    def __post_init__(self) -> None:
        self._check()

    def _check(self) -> None:
        tokens, tiles = self.positions.numel(), self.tile_seq.numel()
        for name, n in (("cu_q", max(1, self.cu_q.numel())), ("positions", tokens), ("tile_seq", tiles),
                        ("tile_q0", tiles), ("counts", 4)):
            _check_ints(name, getattr(self, name), n)
        if self.rows.dtype is not torch.int64:
            raise TypeError("rows must be int64")
        if self.rows.numel() != tokens or not self.rows.is_contiguous():
            raise ValueError("rows must be contiguous with an entry per position")
        if len({t.device for t in (self.cu_q, self.positions, self.rows, self.tile_seq, self.tile_q0,
                                   self.counts)}) > 1:
            raise ValueError("a layout's buffers lie on one device")

    @property
    def _num_seqs(self) -> int:
        return self.cu_q.numel() - 1

    @property
    def _args(self) -> tuple[int, int, int, int, int, int, int, int]:
        """The C call's arguments, of the tensors as they are now. Every call asks: a layout may be a copy, or its
        tensors may have been given other memory."""

        cu_q, positions, rows, tile_seq, tile_q0, counts = (self.cu_q, self.positions, self.rows, self.tile_seq,
                                                            self.tile_q0, self.counts)
        tokens, tiles = positions.numel(), tile_seq.numel()
        if rows.numel() != tokens or tile_q0.numel() != tiles or counts.numel() != 4 or cu_q.dtype is not _I32 \
                or positions.dtype is not _I32 or rows.dtype is not _I64 or tile_seq.dtype is not _I32 \
                or tile_q0.dtype is not _I32 or counts.dtype is not _I32 or not cu_q.is_contiguous() \
                or not positions.is_contiguous() or not rows.is_contiguous() or not tile_seq.is_contiguous() \
                or not tile_q0.is_contiguous() or not counts.is_contiguous():
            self._check()
        return (cu_q.data_ptr(), positions.data_ptr(), rows.data_ptr(), tokens, tile_seq.data_ptr(),
                tile_q0.data_ptr(), tiles, counts.data_ptr())

    @classmethod
    def allocate(cls, num_seqs: int, token_capacity: int, tile_capacity: int,
                 device: torch.device | str) -> "BatchLayout":
        """Buffers for up to ``token_capacity`` tokens and ``tile_capacity`` tiles, parts of one allocation."""

        ends = (2 * token_capacity, 3 * token_capacity, 3 * token_capacity + tile_capacity,
                3 * token_capacity + 2 * tile_capacity, 3 * token_capacity + 2 * tile_capacity + num_seqs + 1)
        buffer = torch.empty(ends[4] + 4, dtype=torch.int32, device=device)
        # Outputs of a step, like those of an op: parts that need no tracking as views of each other.
        rows, positions, tile_seq, tile_q0, cu_q, counts = torch.unsafe_split_with_sizes(
            buffer, (ends[0], token_capacity, tile_capacity, tile_capacity, num_seqs + 1, 4))
        self = object.__new__(cls)  # its buffers are right by construction: checked by the call that uses them
        self.__dict__.update(cu_q=cu_q, positions=positions, rows=rows.view(torch.int64), tile_seq=tile_seq,
                             tile_q0=tile_q0, counts=counts)
        return self


def batch_layout_raw(past: torch.Tensor, lens: torch.Tensor, block_table: torch.Tensor,
                     table_row: torch.Tensor | None, free_blocks: torch.Tensor, block_size: int,
                     layout: BatchLayout) -> None:
    """Launch ``cdb_batch_layout``: block tables, slots and attention tiles of a batch whose request s holds
    ``past[s]`` tokens and brings ``lens[s]`` more. New blocks come from the front of ``free_blocks`` in request
    order and go to the requests' rows of ``block_table``; ``layout`` receives the rest. The caller drops
    ``counts[2]`` ids from its free list and looks at the bits of ``counts[3]``."""

    num_seqs = past.numel()
    if num_seqs > _lib.CDB_LAYOUT_MAX_SEQS:
        raise ValueError(f"a layout takes up to {_lib.CDB_LAYOUT_MAX_SEQS} requests, got {num_seqs}")
    table_rows, width = _check_table(block_table)
    num_free = free_blocks.numel()
    _check_ints("past", past, num_seqs)
    _check_ints("lens", lens, num_seqs)
    _check_ints("free_blocks", free_blocks, num_free)
    if layout._num_seqs != num_seqs:
        raise ValueError(f"the layout holds {layout._num_seqs} requests, got {num_seqs}")
    if table_row is not None:
        _check_ints("table_row", table_row, num_seqs)
    elif table_rows < num_seqs:
        raise ValueError("block_table needs a row per request when table_row is not given")
    _require_here(past, lens, block_table, table_row, free_blocks, layout.cu_q, layout.positions, layout.rows,
                  layout.tile_seq, layout.tile_q0, layout.counts)
    code = _lib.lib().cdb_batch_layout(
        past.data_ptr(), lens.data_ptr(), num_seqs, block_table.data_ptr(), _ptr(table_row), table_rows, width,
        free_blocks.data_ptr(), num_free, block_size, *layout._args, _stream())
    if code:
        _lib.check(code, "cdb_batch_layout")


def _apart(num_seqs: int, tokens: int, tiles: int, device: torch.device) -> tuple[torch.Tensor, ...]:
    """A layout's buffers as tensors of their own, as an op's results have to be."""

    def ints(n: int) -> torch.Tensor:
        return torch.empty(n, dtype=torch.int32, device=device)

    return (ints(num_seqs + 1), ints(tokens), torch.empty(tokens, dtype=torch.int64, device=device), ints(tiles),
            ints(tiles), ints(4))


@torch.library.custom_op("cdb::batch_layout", mutates_args=("block_table",), device_types="cuda")
def batch_layout(past: torch.Tensor, lens: torch.Tensor, block_table: torch.Tensor, table_row: torch.Tensor | None,
                 free_blocks: torch.Tensor, block_size: int, token_capacity: int, tile_capacity: int
                 ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(cu_q, positions, rows, tile_seq, tile_q0, counts) of a batch; see ``batch_layout_raw``."""

    a = _apart(past.numel(), token_capacity, tile_capacity, past.device)
    batch_layout_raw(past, lens, block_table, table_row, free_blocks, block_size, BatchLayout(*a))
    return a


@batch_layout.register_fake
def _(past, lens, block_table, table_row, free_blocks, block_size, token_capacity, tile_capacity):
    return _apart(past.numel(), token_capacity, tile_capacity, past.device)
