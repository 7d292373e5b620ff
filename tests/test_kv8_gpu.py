"""The 8-bit KV cache kernels against the oracle: the write and the codes it leaves exactly, attention within
bounds derived from what each computation rounds."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from continuous_depth_batching_amd import kv8, ops
from oracle import kv8 as oracle
from tests import kv8_helpers as helpers

pytestmark = pytest.mark.gpu
DEV = "cuda"
TINY = 2.0 ** -24  # half a step of fp32


def bounds(kind: str, dtype: str, dim: int, tokens: int) -> dict[str, float]:
    """What a computation rounds, relative (oracle.kv8.attend).

    Scores: dim products summed in fp32 once for each part the query is taken in, and a few roundings of scaling.
    A prefill query in bf16 is its own single part; in fp32 both take three bf16 parts (2^-24 left of each element).
    A bf16 decode query is 3 e4m3 parts, the first with the head's largest element in (224, 448], each next one 16
    times finer: parts of at most 448, 256 and 128 leave at most half their step, 16, 8 and 4, times 16^-(part - 1);
    so 4 / 16^2 of 224, 2^-13.8 of the largest element, after three. Its products sum in fewer bits than fp32: some
    2^-16 of the largest term each, 3 products.
    Probabilities: the exponential and its argument, the fp16 parts they are taken in (2^-11 after one, 2^-22 after
    two for fp32, and 2^-25 at any size), and the fp32 sums over tokens. The result: a half step of its type, and a
    division and a merge in fp32."""
    out = 2.0 ** -8 if dtype == "bf16" else 8 * TINY
    prob = 2.0 ** -11 if dtype == "bf16" else 2.0 ** -22
    if kind == "decode":
        parts, left, top = (3, 0.0, 2.0 ** -13.8 + 3 * 2.0 ** -16) if dtype == "bf16" else (3, TINY, 0.0)
    else:
        parts, left, top = (1, 0.0, 0.0) if dtype == "bf16" else (3, TINY, 0.0)
    return dict(round_off=out + 8 * TINY, score_off=(parts * dim + 8) * TINY + left, top_off=top,
                prob_off=prob + (2 * tokens + 16) * TINY, floor=2.0 ** -25)


def dev(a, dtype=None) -> torch.Tensor:
    t = torch.from_numpy(np.ascontiguousarray(a)) if isinstance(a, np.ndarray) else torch.as_tensor(a)
    return (t if dtype is None else t.to(dtype)).to(DEV)


def f32(t: torch.Tensor | None) -> np.ndarray | None:
    return None if t is None else t.float().cpu().numpy()


# -- write ---------------------------------------------------------------------------------------------------------


class WriteCase:
    def __init__(self, seed, dtype, heads, kv, dim, style, bias, block, seqs, *, layers=2, pad=0, std=1.0, nan=False):
        """seqs: (cached tokens, new tokens) a sequence."""
        rng = np.random.default_rng(seed)
        past, new = np.array([p for p, _ in seqs]), np.array([n for _, n in seqs])
        table, blocks = helpers.tables(rng, past + new, block)
        self.pool, self.cache = helpers.random_pool(rng, layers, blocks, block, kv, dim, DEV, nan_codes=nan)
        pos = np.concatenate([np.arange(p, p + n) for p, n in seqs])
        rows = np.concatenate([helpers.slots(table[s], np.arange(p, p + n), block) for s, (p, n) in enumerate(seqs)])
        self.rows, self.pos = np.concatenate([rows, np.full(pad, -1)]), np.concatenate([pos, np.full(pad, -1)])
        tokens = self.rows.size
        self.cos, self.sin = helpers.rope_tables(dim, int(pos.max()) + 1) if style else (None, None)
        self.style, self.layer, self.dim = style, layers - 1, dim
        fused = helpers.values(rng, dtype, tokens, (heads + 2 * kv) * dim, std=std).to(DEV)
        self.q = fused[:, :heads * dim].view(tokens, heads, dim)
        self.k = fused[:, heads * dim:(heads + kv) * dim].view(tokens, kv, dim)
        self.v = fused[:, (heads + kv) * dim:].view(tokens, kv, dim)
        self.q_bias = helpers.values(rng, dtype, heads, dim, std=0.1).to(DEV) if bias else None
        self.k_bias = helpers.values(rng, dtype, kv, dim, std=0.1).to(DEV) if bias else None

    def run(self, q_out=None, **over):
        a = dict(q=self.q, k=self.k, v=self.v, rows=dev(self.rows), pos=dev(self.pos, torch.int32)) | over
        q_out = torch.full(self.q.shape, 7.0, dtype=self.q.dtype, device=DEV) if q_out is None else q_out
        kv8.write_raw(a["q"], a["k"], a["v"], q_out if a["q"] is not None else None, self.pool, self.layer, a["rows"],
                      a["pos"], None if self.cos is None else dev(self.cos),
                      None if self.sin is None else dev(self.sin),
                      self.style, self.q_bias if a["q"] is not None else None, self.k_bias)
        return q_out

    def expect(self):
        pos = np.maximum(self.pos, 0)
        k = oracle.rotate(f32(self.k), f32(self.k_bias), self.cos, self.sin, pos, self.style)
        self.cache.write(self.layer, self.rows, k, f32(self.v))
        q = oracle.rotate(f32(self.q), f32(self.q_bias), self.cos, self.sin, pos, self.style)
        return torch.from_numpy(q).to(self.q.dtype)

    def check(self):
        got, want = self.run().cpu(), self.expect()
        live = torch.from_numpy(self.rows >= 0)
        assert torch.equal(got[live], want[live])
        assert (got[~live] == 7.0).all()  # padding tokens keep what was there
        helpers.same_cache(self.pool, self.cache)


SEQS = {
    "single": [(0, 1)],
    "edges": [(0, 16), (0, 15), (0, 17), (15, 1), (15, 2), (16, 16), (1, 15), (7, 40), (3, 1)],
    "decode": [(i * 7, 1) for i in range(40)],
    "prompt": [(0, 700), (130, 500)],
}


@pytest.mark.parametrize("seqs", sorted(SEQS))
@pytest.mark.parametrize("dtype,heads,kv,dim,style,bias,block", [
    ("bf16", 4, 4, 128, 1, False, 16), ("bf16", 8, 2, 64, 2, True, 32), ("f32", 5, 5, 96, 1, True, 64),
    ("bf16", 3, 1, 96, 2, False, 16), ("f32", 4, 2, 128, 0, False, 16), ("f32", 2, 2, 64, 1, True, 16),
    ("bf16", 2, 2, 96, 1, True, 128),
])
def test_write_codes_and_rotates(seqs, dtype, heads, kv, dim, style, bias, block) -> None:
    WriteCase(1, dtype, heads, kv, dim, style, bias, block, SEQS[seqs], pad=3).check()


@pytest.mark.parametrize("std", [1e-3, 300.0, 1e30])
def test_write_scales_grow_and_hold(std) -> None:
    """Small values under a larger scale, and values that make a tile's scale grow."""
    WriteCase(2, "bf16", 2, 2, 64, 1, False, 16, [(5, 3), (9, 30), (0, 4)], std=std).check()


def test_write_keeps_infinities_and_nan_apart() -> None:
    c = WriteCase(3, "f32", 2, 2, 64, 0, False, 16, [(3, 20), (0, 5)], nan=True)
    c.k[4, 0, 3], c.k[5, 1, 60], c.v[6, 0, 1], c.v[20, 1, 0] = float("inf"), float("nan"), float("-inf"), float("nan")
    c.k[21, 0] = float("nan")  # a token with nothing finite
    c.check()


def test_write_zeros() -> None:
    c = WriteCase(4, "bf16", 2, 2, 64, 1, False, 16, [(0, 20), (4, 2)])
    c.k.zero_()
    c.v.zero_()
    c.check()


def test_write_many_single_tokens_and_prompts_together() -> None:
    """More tokens than one wave takes each: chunks of 16 in which every token may start a tile."""
    rng = np.random.default_rng(5)
    seqs = [(int(p), 1) for p in rng.integers(0, 50, size=900)] + [(3, 150), (0, 33)]
    WriteCase(5, "bf16", 1, 1, 64, 1, False, 16, seqs).check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("style", [0, 1, 2])
def test_write_of_unaligned_views(dtype, style) -> None:
    """Token strides and bases that no 16-byte load fits."""
    c = WriteCase(6, dtype, 3, 2, 96, style, True, 16, [(2, 19), (0, 3)])
    tokens = c.k.shape[0]
    wide = torch.zeros(tokens, 7 * 96 + 3, dtype=c.k.dtype, device=DEV)
    q, k, v = (wide[:, at * 96 + 1:(at + n) * 96 + 1].view(tokens, n, 96) for at, n in ((0, 3), (3, 2), (5, 2)))
    q.copy_(c.q), k.copy_(c.k), v.copy_(c.v)
    got, want = c.run(q=q, k=k, v=v).cpu(), c.expect()
    assert torch.equal(got, want)
    helpers.same_cache(c.pool, c.cache)


def test_write_of_keys_and_values_alone() -> None:
    c = WriteCase(7, "bf16", 2, 2, 128, 1, True, 16, [(0, 40)])
    c.run(q=None)
    c.expect()
    helpers.same_cache(c.pool, c.cache)


def test_write_skips_slots_and_positions_out_of_range() -> None:
    c = WriteCase(8, "bf16", 2, 2, 64, 1, False, 16, [(0, 20)])
    rows, pos = c.rows.copy(), c.pos.copy()
    rows[17] = c.pool.num_blocks * 16   # past the pool: no key, but a query
    pos[18] = 20                        # past the tables
    pos[19] = -3
    got = c.run(rows=dev(rows), pos=dev(pos, torch.int32)).cpu()
    c.rows[17:] = -1
    want = c.expect()
    assert torch.equal(got[:18], want[:18]) and got[18:].isnan().all()
    helpers.same_cache(c.pool, c.cache)


def test_write_op_returns_rotated_queries() -> None:
    c = WriteCase(9, "bf16", 4, 2, 64, 1, False, 16, [(0, 20)], pad=2)
    got = torch.ops.cdb.kv8_write(c.q, c.k, c.v, c.pool.codes, c.pool.scales, c.layer, dev(c.rows),
                                  dev(c.pos, torch.int32), dev(c.cos), dev(c.sin), 1, None, None).cpu()
    want = c.expect()
    assert torch.equal(got[:20], want[:20]) and (got[20:] == 0).all()
    helpers.same_cache(c.pool, c.cache)


# -- decode --------------------------------------------------------------------------------------------------------


class DecodeCase:
    def __init__(self, seed, dtype, heads, kv, dim, style, bias, block, contexts, *, layers=3, nan=False, std=1.0,
                 by_row=False, longest=None):
        """contexts: tokens a row attends over, its new one included (0: padding row)."""
        rng = np.random.default_rng(seed)
        self.contexts = np.array(contexts)
        n = len(contexts)
        table, blocks = helpers.tables(rng, self.contexts, block)
        self.block, self.dtype, self.dim, self.style = block, dtype, dim, style
        self.table_row = None
        if by_row:
            order = rng.permutation(n + 2)
            wide = np.full((n + 2, table.shape[1]), -1, np.int32)
            wide[order[:n]] = table
            table, self.table_row = wide, order[:n].astype(np.int32)
        self.table = table
        # NaN codes only where no row looks: behind the contexts, and in spare blocks.
        self.pool, self.cache = helpers.random_pool(rng, layers, blocks, block, kv, dim, DEV)
        if nan:
            seen = np.zeros((blocks * block), bool)
            for b in range(n):
                seen[self.slots(b, np.arange(max(self.contexts[b] - 1, 0)))] = True
            hide = ~seen.reshape(-1, 16)
            self.cache.codes = np.where(hide[None, None, :, None, :, None], np.nan, self.cache.codes)
            self.pool.codes.copy_(helpers.pack(self.cache.codes, block).to(DEV))
        self.layer = rng.integers(0, layers, size=n).astype(np.int32)
        self.pos = (self.contexts - 1).astype(np.int32)
        self.cos, self.sin = helpers.rope_tables(dim, int(self.contexts.max()) + 1) if style else (None, None)
        fused = helpers.values(rng, dtype, n, (heads + 2 * kv) * dim, std=std).to(DEV)
        self.q = fused[:, :heads * dim].view(n, heads, dim)
        self.k = fused[:, heads * dim:(heads + kv) * dim].view(n, kv, dim)
        self.v = fused[:, (heads + kv) * dim:].view(n, kv, dim)
        self.q_bias = helpers.values(rng, dtype, heads, dim, std=0.1).to(DEV) if bias else None
        self.k_bias = helpers.values(rng, dtype, kv, dim, std=0.1).to(DEV) if bias else None
        self.scale = dim ** -0.5
        self.workspace = torch.empty(kv8.decode_workspace_bytes(n, heads, kv, dim, longest or int(self.contexts.max())),
                                     dtype=torch.uint8, device=DEV)

    def slots(self, b, positions):
        row = self.table[b if self.table_row is None else self.table_row[b]]
        return helpers.slots(row, positions, self.block)

    def args(self, **over):
        a = dict(q=self.q, k=self.k, v=self.v, pool=self.pool, layer=dev(self.layer), layer0=0, table=dev(self.table),
                 table_row=None if self.table_row is None else dev(self.table_row), pos=dev(self.pos),
                 cos=None if self.cos is None else dev(self.cos), sin=None if self.sin is None else dev(self.sin),
                 style=self.style, q_bias=self.q_bias, k_bias=self.k_bias,
                 out=torch.full(self.q.shape, 7.0, dtype=self.q.dtype, device=DEV), ws=self.workspace, scale=self.scale)
        return a | over

    def run(self, **over):
        return kv8.decode_attention_raw(*self.args(**over).values())

    def expect(self, rows=None):
        pos = np.maximum(self.pos, 0)
        k = oracle.rotate(f32(self.k), f32(self.k_bias), self.cos, self.sin, pos, self.style)
        q = oracle.rotate(f32(self.q), f32(self.q_bias), self.cos, self.sin, pos, self.style).astype(np.float64)
        want, bound = np.zeros(q.shape), np.zeros(q.shape)
        for b in range(len(pos)) if rows is None else rows:
            if self.pos[b] < 0:
                continue
            at = self.slots(b, np.arange(self.pos[b] + 1))
            self.cache.append(self.layer[b], int(at[-1]), k[b:b + 1], f32(self.v)[b:b + 1])
            keys, vals = (self.cache.values(self.layer[b], plane, at) for plane in (0, 1))
            want[b:b + 1], bound[b:b + 1] = oracle.attend(q[b:b + 1], keys, vals, self.pos[b:b + 1], self.scale,
                                                          **bounds("decode", self.dtype, self.dim, self.pos[b] + 1))
        return want, bound

    def check(self):
        got = self.run()
        helpers.close(got, *self.expect())
        helpers.same_cache(self.pool, self.cache)


CONTEXTS = [1, 2, 15, 16, 17, 32, 33, 64, 65, 129, 255, 256, 257, 300, 513, 900, 0, 1100]


@pytest.mark.parametrize("dtype,heads,kv,dim,style,bias,block", [
    ("bf16", 4, 4, 128, 1, False, 16), ("bf16", 8, 2, 64, 2, True, 32), ("bf16", 5, 5, 96, 2, True, 16),
    ("f32", 3, 3, 64, 1, False, 16), ("f32", 4, 2, 128, 1, True, 64), ("f32", 2, 1, 96, 0, False, 16),
    ("bf16", 14, 2, 128, 0, False, 128), ("bf16", 16, 1, 96, 1, True, 16), ("f32", 6, 3, 96, 1, False, 16),
    ("f32", 2, 2, 128, 2, False, 16),
])
def test_decode_matches_the_definition(dtype, heads, kv, dim, style, bias, block) -> None:
    DecodeCase(11, dtype, heads, kv, dim, style, bias, block, CONTEXTS, nan=True).check()


@pytest.mark.parametrize("heads,kv", [(17, 1), (20, 1), (40, 2), (64, 1)])
def test_decode_with_more_than_16_query_heads_a_kv_head(heads, kv) -> None:
    DecodeCase(12, "bf16", heads, kv, 64, 1, False, 16, [1, 16, 40, 300, 530], nan=True).check()


@pytest.mark.parametrize("std", [1e-4, 30.0, 300.0])
def test_decode_scales_grow_and_hold(std) -> None:
    """A new token far below the tile's scale, and one that makes it grow (with large scores among small ones)."""
    DecodeCase(13, "bf16", 2, 2, 64, 1, False, 16, [1, 2, 5, 16, 17, 18, 31, 270, 272, 273], std=std).check()


@pytest.mark.parametrize("dtype,heads,kv,dim", [("bf16", 4, 2, 128), ("f32", 1, 1, 64), ("bf16", 20, 1, 96)])
def test_decode_chunk_edges(dtype, heads, kv, dim) -> None:
    """Contexts around the length of a chunk and of two, and rows of several chunks beside rows of one."""
    contexts = [1009, 1023, 1024, 1025, 1040, 1041, 2047, 2048, 2049, 5, 4000]
    DecodeCase(26, dtype, heads, kv, dim, 1, False, 16, contexts, nan=True).check()


def test_decode_over_permuted_table_rows() -> None:
    DecodeCase(14, "bf16", 4, 2, 128, 1, False, 32, [1, 70, 0, 300, 17], by_row=True, nan=True).check()


def test_decode_long_context_and_short_workspace() -> None:
    """Partials for fewer chunks than the context has: the chunks lengthen, past one look-up window too."""
    for longest in (300, 2048, 5000):
        DecodeCase(15, "bf16", 2, 1, 64, 1, False, 16, [5000, 100, 4097], longest=longest, nan=True).check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_context_of_more_chunks_than_a_row_has(dtype) -> None:
    """Past 64 chunks of 1024 tokens a row takes longer ones, with a workspace of any size."""
    DecodeCase(18, dtype, 2, 1, 64, 1, False, 64, [70_000, 3, 65_537], layers=1).check()


def test_decode_marks_rows_out_of_range() -> None:
    c = DecodeCase(16, "bf16", 2, 2, 64, 1, False, 16, [20, 300, 40, 50, 60, 300, 33], by_row=True)
    c.table[c.table_row[1], 3] = c.pool.num_blocks     # a block past the pool inside the context
    c.table[c.table_row[5], 18] = -1                   # the last block, where the row would append
    c.layer[2] = 3
    rows = c.table_row.copy()
    rows[3] = c.table.shape[0]
    rows[4] = -1
    c.table_row, keep = rows, c.table_row
    got = c.run()
    c.table_row = keep
    assert got[1:6].isnan().all()
    fine = [0, 6]
    want, bound = c.expect(fine)
    helpers.close(got[fine], want[fine], bound[fine])
    # Row 1 appends to a sound block all the same; the others leave the cache alone.
    k = oracle.rotate(f32(c.k), None, c.cos, c.sin, np.maximum(c.pos, 0), 1)
    c.cache.append(c.layer[1], int(c.slots(1, np.array([299]))[0]), k[1:2], f32(c.v)[1:2])
    helpers.same_cache(c.pool, c.cache)


def test_decode_marks_positions_past_the_tables() -> None:
    c = DecodeCase(17, "bf16", 2, 2, 64, 1, False, 16, [20, 40])
    pos = c.pos.copy()
    pos[0] = c.table.shape[1] * 16
    before = c.pool.codes.view(torch.uint8).clone()
    got = c.run(pos=dev(pos), cos=dev(c.cos[:30]), sin=dev(c.sin[:30]))
    assert got.isnan().all() and torch.equal(before, c.pool.codes.view(torch.uint8))


def test_decode_nan_of_a_seen_key_or_value() -> None:
    c = DecodeCase(18, "bf16", 2, 1, 64, 0, False, 16, [40, 40, 40])
    for b, plane in ((0, 0), (1, 1)):
        slot = int(c.slots(b, np.array([7]))[0])
        c.cache.codes[c.layer[b], plane, slot // 16, 0, slot % 16, 5] = np.nan
    c.pool.codes.copy_(helpers.pack(c.cache.codes, 16).to(DEV))
    got = c.run().float().cpu().numpy()
    assert np.isnan(got[0]).all()                      # a key: every score of the row
    assert np.isnan(got[1][:, 5]).all() and np.isnan(got[1]).sum() == 2  # a value: its element alone
    want, bound = c.expect([2])
    helpers.close(torch.from_numpy(got[2:]), want[2:], bound[2:])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("style,dim", [(0, 64), (1, 96), (2, 128)])
def test_decode_of_unaligned_views(dtype, style, dim) -> None:
    c = DecodeCase(19, dtype, 3, 1, dim, style, True, 16, [1, 40, 300])
    wide = torch.zeros(3, 5 * dim + 3, dtype=c.q.dtype, device=DEV)
    q, k, v = (wide[:, at * dim + 1:(at + n) * dim + 1].view(3, n, dim) for at, n in ((0, 3), (3, 1), (4, 1)))
    q.copy_(c.q), k.copy_(c.k), v.copy_(c.v)
    helpers.close(c.run(q=q, k=k, v=v), *c.expect())
    helpers.same_cache(c.pool, c.cache)


def test_decode_row_is_bit_identical_in_any_batch() -> None:
    contexts = [700, 3, 257, 1500, 64, 16, 300]
    c = DecodeCase(20, "bf16", 8, 2, 128, 1, False, 16, contexts)
    whole = c.run()
    for rows in ([3], [0, 6], [6, 5, 4, 3, 2, 1, 0]):
        r = torch.tensor(rows, device=DEV)
        a = c.args()
        part = c.run(q=c.q[r], k=c.k[r], v=c.v[r], layer=a["layer"][r], table=a["table"][r], pos=a["pos"][r],
                     out=torch.empty_like(whole[r]))
        assert torch.equal(part, whole[r])


def test_decode_layer_base_without_row_offsets() -> None:
    c = DecodeCase(21, "bf16", 2, 2, 64, 1, False, 16, [20, 300])
    c.layer[:] = 2
    helpers.close(c.run(layer=None, layer0=2), *c.expect())
    helpers.same_cache(c.pool, c.cache)


def test_decode_graph_replays_and_streams() -> None:
    """A captured launch replayed between eager work, and launches on two streams with a workspace each."""
    c = DecodeCase(22, "bf16", 4, 2, 128, 1, False, 16, [700, 3, 257, 1500])
    a = c.args()
    want = c.run(**{k: a[k] for k in ("out",)}).clone()  # appends once; the same append again changes nothing
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv8.decode_attention_raw(*a.values())
    for _ in range(3):
        a["out"].fill_(3.0)
        c.workspace.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a["out"], want)
    side = torch.cuda.Stream()
    other = c.args(ws=torch.empty_like(c.workspace))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv8.decode_attention_raw(*other.values())
    again = c.run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, want) and torch.equal(other["out"], want)


def test_decode_op() -> None:
    c = DecodeCase(23, "bf16", 4, 2, 128, 1, False, 16, [700, 3, 0])
    a = c.args()
    got = torch.ops.cdb.kv8_decode_attention(c.q, c.k, c.v, c.pool.codes, c.pool.scales, a["layer"], 0, a["table"],
                                             None,
                                             a["pos"], a["cos"], a["sin"], 1, None, None, c.workspace, c.scale)
    helpers.close(got, *c.expect())
    assert (got[2] == 0).all()


def test_calls_refuse_tensors_on_the_cpu() -> None:
    c = DecodeCase(24, "bf16", 2, 2, 64, 1, False, 16, [20])
    with pytest.raises(RuntimeError, match="GPU only"):
        c.run(pos=torch.from_numpy(c.pos))


def test_decode_empty_batch() -> None:
    c = DecodeCase(25, "bf16", 2, 2, 64, 1, False, 16, [20])
    a = c.args()
    z = torch.zeros(0, dtype=torch.int32, device=DEV)
    out = c.run(q=c.q[:0], k=c.k[:0], v=c.v[:0], layer=z, pos=z, out=torch.empty_like(c.q[:0]), table=a["table"])
    assert out.shape == (0, 2, 64)


# -- prefill -------------------------------------------------------------------------------------------------------


class PrefillCase:
    def __init__(self, seed, dtype, heads, kv, dim, block, seqs, *, layers=2, nan=False, std=1.0):
        rng = np.random.default_rng(seed)
        self.past, self.new = np.array([p for p, _ in seqs]), np.array([n for _, n in seqs])
        self.block, self.dtype, self.dim = block, dtype, dim
        self.table, blocks = helpers.tables(rng, self.past + self.new, block)
        self.pool, self.cache = helpers.random_pool(rng, layers, blocks, block, kv, dim, DEV)
        if nan:
            seen = np.zeros((blocks * block), bool)
            for s in range(len(seqs)):
                seen[helpers.slots(self.table[s], np.arange(self.past[s] + self.new[s]), block)] = True
            self.cache.codes = np.where(~seen.reshape(-1, 16)[None, None, :, None, :, None], np.nan, self.cache.codes)
            self.upload()
        self.layer = layers - 1
        self.cu = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.q = helpers.values(rng, dtype, int(self.cu[-1]), heads, dim, std=std).to(DEV)
        self.scale = dim ** -0.5

    def upload(self):
        self.pool.codes.copy_(helpers.pack(self.cache.codes, self.block).to(DEV))

    def run(self, splits=1, extra_tiles=0, **over):
        seq, q0 = ops.prefill_tiles(self.new, self.past)
        seq = np.concatenate([seq, np.full(extra_tiles, -1, np.int32)])
        q0 = np.concatenate([q0, np.zeros(extra_tiles, np.int32)])
        heads = self.q.shape[1]
        ws = torch.full((kv8.prefill_workspace_bytes(len(seq), splits, heads, self.dim),), 255, dtype=torch.uint8,
                        device=DEV)
        a = dict(q=self.q, pool=self.pool, layer=self.layer, table=dev(self.table),
                 table_row=dev(np.arange(len(self.past), dtype=np.int32)), cu=dev(self.cu),
                 past=dev(self.past.astype(np.int32)), seq=dev(seq), q0=dev(q0),
                 out=torch.full(self.q.shape, 7.0, dtype=self.q.dtype, device=DEV), scale=self.scale, splits=splits,
                 ws=ws if splits > 1 else None) | over
        return kv8.prefill_attention_raw(*a.values())

    def expect(self, seqs=None):
        q = self.q.cpu().double().numpy()
        want, bound = np.zeros(q.shape), np.zeros(q.shape)
        for s in range(len(self.past)) if seqs is None else seqs:
            n, p = int(self.new[s]), int(self.past[s])
            at = helpers.slots(self.table[s], np.arange(p + n), self.block)
            keys, vals = (self.cache.values(self.layer, plane, at) for plane in (0, 1))
            mine = slice(self.cu[s], self.cu[s + 1])
            want[mine], bound[mine] = oracle.attend(q[mine], keys, vals, p + np.arange(n), self.scale,
                                                    **bounds("prefill", self.dtype, self.dim, p + n))
        return want, bound


PREFILLS = {
    "short": [(0, 1), (0, 2), (0, 16), (0, 17), (0, 31), (0, 32), (0, 33)],
    "tiles": [(0, 127), (0, 128), (0, 129), (0, 260)],
    "history": [(5, 3), (100, 40), (15, 1), (1000, 30), (33, 130)],
    "empty": [(0, 5), (40, 0), (0, 0), (3, 20)],
}


@pytest.mark.parametrize("seqs", sorted(PREFILLS))
@pytest.mark.parametrize("dtype,heads,kv,dim,block", [
    ("bf16", 2, 2, 128, 16), ("bf16", 4, 1, 64, 32), ("bf16", 3, 3, 96, 16), ("f32", 2, 1, 128, 16),
    ("f32", 2, 2, 64, 64), ("f32", 2, 2, 96, 16),
])
def test_prefill_matches_the_definition(seqs, dtype, heads, kv, dim, block) -> None:
    c = PrefillCase(31, dtype, heads, kv, dim, block, PREFILLS[seqs], nan=True)
    helpers.close(c.run(extra_tiles=2), *c.expect())


@pytest.mark.parametrize("splits", [2, 3, 7])
@pytest.mark.parametrize("dtype,heads,kv,dim", [("bf16", 4, 2, 128), ("f32", 2, 2, 64), ("bf16", 2, 2, 96)])
def test_prefill_split_key_ranges(splits, dtype, heads, kv, dim) -> None:
    c = PrefillCase(32, dtype, heads, kv, dim, 16, [(1000, 30), (0, 200), (300, 129), (0, 1)], nan=True)
    helpers.close(c.run(splits=splits, extra_tiles=1), *c.expect())


@pytest.mark.parametrize("std", [0.01, 8.0])
def test_prefill_of_flat_and_peaked_scores(std) -> None:
    c = PrefillCase(33, "bf16", 2, 2, 128, 16, [(200, 140)], std=std)
    helpers.close(c.run(), *c.expect())


def test_prefill_values_whose_scales_differ() -> None:
    """Tiles of tiny and huge values next to each other, the larger ones coming first, last and between."""
    c = PrefillCase(34, "bf16", 2, 2, 64, 16, [(100, 60), (0, 200)])
    rng = np.random.default_rng(35)
    e = rng.integers(-40, 20, size=c.cache.exponents.shape)
    c.cache.exponents[:, 1] = e[:, 1]
    nt = c.block // 16
    e_bytes = torch.from_numpy((c.cache.exponents + 127).astype(np.uint8))
    layers, _, tiles, kv = e_bytes.shape
    c.pool.scales.copy_(e_bytes.view(layers, 2, tiles // nt, nt, kv).transpose(3, 4))
    helpers.close(c.run(), *c.expect())


def test_prefill_sequence_out_of_range_gives_nan() -> None:
    c = PrefillCase(36, "bf16", 2, 2, 64, 16, [(0, 40), (30, 40), (0, 50), (0, 20)])
    c.table[0, 1] = c.pool.num_blocks
    c.table[2, 0] = -1
    for splits in (1, 2):
        rows = np.arange(4, dtype=np.int32)
        rows[3] = 4
        got = c.run(splits=splits, table_row=dev(rows))
        assert got[:40].isnan().all() and got[80:].isnan().all()
        want, bound = c.expect([1])
        helpers.close(got[40:80], want[40:80], bound[40:80])


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("bf16", 96), ("f32", 64)])
def test_prefill_nan_values_reach_only_queries_that_see_them(dtype, dim) -> None:
    """NaN codes of keys and values inside the chunk and in its history: earlier queries are untouched, later ones
    have NaN (a key: everywhere; a value: in its element)."""
    c = PrefillCase(39, dtype, 2, 2, dim, 16, [(40, 90), (0, 70)])
    for s, at, plane, head, d in ((0, 60, 1, 0, 5), (0, 61, 1, 0, 6), (0, 100, 1, 1, dim - 1), (1, 33, 0, 0, 3),
                                  (1, 3, 1, 1, 9)):
        slot = int(helpers.slots(c.table[s], np.array([at]), 16)[0])
        c.cache.codes[c.layer, plane, slot // 16, head, slot % 16, d] = np.nan
    c.upload()
    for splits in (1, 3):
        got = c.run(splits=splits).float().cpu().numpy()
        hit = np.zeros(got.shape, bool)
        hit[60 - 40:90, 0, 5] = hit[61 - 40:90, 0, 6] = hit[100 - 40:90, 1, dim - 1] = True
        hit[90 + 33:, 0, :] = True
        hit[90 + 3:, 1, 9] = True
        np.testing.assert_array_equal(np.isnan(got), hit)
        c.cache.codes, keep = np.nan_to_num(c.cache.codes), c.cache.codes
        want, bound = c.expect()
        c.cache.codes = keep
        ok = np.abs(got - want) <= bound
        assert ok[:60 - 40].all() and ok[90:90 + 3].all() and ok[90:90 + 33, 0].all()


def test_prefill_graph_replays() -> None:
    c = PrefillCase(37, "bf16", 2, 1, 128, 16, [(700, 60), (0, 200)])
    seq, q0 = ops.prefill_tiles(c.new, c.past)
    ws = torch.empty(kv8.prefill_workspace_bytes(len(seq), 3, 2, 128), dtype=torch.uint8, device=DEV)
    out = torch.empty_like(c.q)
    args = (c.q, c.pool, c.layer, dev(c.table), dev(np.arange(2, dtype=np.int32)), dev(c.cu),
            dev(c.past.astype(np.int32)), dev(seq), dev(q0), out, c.scale, 3, ws)
    kv8.prefill_attention_raw(*args)
    want = out.clone()
    helpers.close(want, *c.expect())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv8.prefill_attention_raw(*args)
    for _ in range(3):
        out.fill_(3.0)
        ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_prefill_op() -> None:
    c = PrefillCase(38, "bf16", 4, 2, 64, 16, [(20, 60)])
    seq, q0 = ops.prefill_tiles(c.new, c.past)
    got = torch.ops.cdb.kv8_prefill_attention(c.q, c.pool.codes, c.pool.scales, c.layer, dev(c.table),
                                              dev([0], torch.int32), dev(c.cu), dev(c.past.astype(np.int32)),
                                              dev(seq), dev(q0), c.scale, 1, None)
    helpers.close(got, *c.expect())


# -- layout --------------------------------------------------------------------------------------------------------


def plain_layout(past, lens, table, rows, free, block):
    """cu_q, positions, slots, tiles (longest key range first) and the table, one request after the other."""
    cu, pos, slot, tiles, taken = [0], [], [], [], 0
    table = table.copy()
    for s, (p, n) in enumerate(zip(past, lens)):
        for col in range(-(-p // block), -(-(p + n) // block)):
            table[rows[s], col] = free[taken] if taken < len(free) else -1
            taken += 1
        for t in range(p, p + n):
            b = table[rows[s], t // block]
            pos.append(t)
            slot.append(b * block + t % block if b >= 0 else -1)
        cu.append(cu[-1] + n)
        tiles += [(p + min(q + 128, n), s, q) for q in range(0, n, 128)]
    tiles.sort(key=lambda t: -t[0])
    return cu, pos, slot, [(s, q) for _, s, q in tiles], taken, table


def run_layout(past, lens, table, rows, free, block, tokens, tiles):
    out = kv8.BatchLayout.allocate(len(past), tokens, tiles, DEV)
    t = dev(table)
    kv8.batch_layout_raw(dev(past, torch.int32), dev(lens, torch.int32), t,
                         None if rows is None else dev(rows, torch.int32),
                         dev(free, torch.int32), block, out)
    return out, t.cpu().numpy()


@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("seqs,hi,past_hi", [(1, 1, 0), (1, 5000, 300), (7, 200, 0), (33, 300, 900), (1500, 5, 40),
                                             (4000, 2, 3), (64, 1, 700)])
def test_layout_matches_the_requests_one_by_one(block, seqs, hi, past_hi) -> None:
    rng = np.random.default_rng(41)
    lens, past = rng.integers(0 if seqs > 1 else hi, hi + 1, size=seqs), rng.integers(0, past_hi + 1, size=seqs)
    width = -(-(past_hi + hi) // block) + 1
    rows = rng.permutation(seqs + 2)[:seqs]
    table = rng.integers(0, 1000, size=(seqs + 2, width)).astype(np.int32)
    need = int((-(-(past + lens) // block) - -(-past // block)).sum())
    free = rng.permutation(need + 5).astype(np.int32)
    total, tiles = int(lens.sum()), int((-(-lens // 128)).sum())
    out, got_table = run_layout(past, lens, table, rows, free, block, total + 3, tiles + 4)
    cu, pos, slot, order, taken, want_table = plain_layout(past, lens, table, rows, free, block)
    assert out.counts.tolist() == [total, tiles, taken, 0]
    assert out.cu_q.tolist() == cu
    assert out.positions.tolist() == pos + [-1] * 3 and out.rows.tolist() == slot + [-1] * 3
    assert out.tile_seq.tolist() == [s for s, _ in order] + [-1] * 4
    assert out.tile_q0.tolist() == [q for _, q in order] + [0] * 4
    np.testing.assert_array_equal(got_table, want_table)


def test_layout_without_requests_or_tokens() -> None:
    table = np.zeros((2, 3), np.int32)
    for past, lens in (([], []), ([5, 0], [0, 0])):
        out, got = run_layout(np.array(past, np.int32), np.array(lens, np.int32), table, None, np.zeros(0, np.int32),
                              16,
                              4, 2)
        assert out.counts.tolist() == [0, 0, 0, 0] and out.cu_q.tolist() == [0] * (len(past) + 1)
        assert out.rows.tolist() == [-1] * 4 and out.tile_seq.tolist() == [-1] * 2
        np.testing.assert_array_equal(got, table)


def test_layout_op() -> None:
    past, lens, table = np.array([0, 20]), np.array([40, 150]), np.full((2, 12), 99, np.int32)
    free = np.arange(20, dtype=np.int32)
    t = dev(table)
    cu, pos, slot, seq, q0, counts = torch.ops.cdb.batch_layout(dev(past, torch.int32), dev(lens, torch.int32), t, None,
                                                                dev(free), 16, 190, 3)
    want = plain_layout(past, lens, table, [0, 1], free, 16)
    assert (cu.tolist(), pos.tolist(), slot.tolist()) == want[:3]
    assert list(zip(seq.tolist(), q0.tolist())) == want[3] and counts.tolist() == [190, 3, want[4], 0]
    np.testing.assert_array_equal(t.cpu().numpy(), want[5])


def test_layout_reports_what_does_not_fit() -> None:
    past, lens = np.array([0, 20]), np.array([40, 150])
    table = np.full((2, 12), 99, np.int32)
    free = np.array([4, 5, 6, 7], np.int32)
    out, got = run_layout(past, lens, table, None, free, 16, 50, 2)
    assert out.counts.tolist() == [190, 3, 12, kv8.LAYOUT_TOKENS_FULL | kv8.LAYOUT_TILES_FULL | kv8.LAYOUT_NO_BLOCKS]
    cu, pos, slot, order, _, want = plain_layout(past, lens, table, [0, 1], free, 16)
    assert out.positions.tolist() == pos[:50] and out.rows.tolist() == slot[:50]
    assert out.tile_seq.tolist() == [s for s, _ in order[:2]]
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("seqs", [255, 256, 257, 1000, 1024, 1025])
def test_layout_at_the_sizes_where_its_scan_changes(seqs) -> None:
    rng = np.random.default_rng(42)
    lens, past = rng.integers(0, 300, size=seqs), rng.integers(0, 200, size=seqs)
    lens[[0, seqs // 2, -1]] = 0, 129, 300
    table = rng.integers(0, 1000, size=(seqs, 32)).astype(np.int32)
    free = rng.permutation(seqs * 32).astype(np.int32)
    total, tiles = int(lens.sum()), int((-(-lens // 128)).sum())
    out, got_table = run_layout(past, lens, table, None, free, 16, total, tiles)
    cu, pos, slot, order, taken, want_table = plain_layout(past, lens, table, np.arange(seqs), free, 16)
    assert out.counts.tolist() == [total, tiles, taken, 0]
    assert out.cu_q.tolist() == cu and out.positions.tolist() == pos and out.rows.tolist() == slot
    assert list(zip(out.tile_seq.tolist(), out.tile_q0.tolist())) == order
    np.testing.assert_array_equal(got_table, want_table)


def test_layout_of_too_many_tokens_to_count_is_left_out() -> None:
    lens = np.full(3, 1 << 30)
    table = np.full((3, 1 << 14), 7, np.int32)
    out, got_table = run_layout(np.zeros(3), lens, table, None, np.arange(5), 1 << 16, 40, 9)
    assert out.counts.tolist() == [2 ** 31 - 1, 3 << 23, 3 << 14, kv8.LAYOUT_TOKENS_FULL | kv8.LAYOUT_TILES_FULL |
                                   kv8.LAYOUT_NO_BLOCKS]
    assert out.positions.tolist() == [-1] * 40 and out.rows.tolist() == [-1] * 40
    assert out.tile_seq.tolist() == [-1] * 9 and out.tile_q0.tolist() == [0] * 9
    np.testing.assert_array_equal(got_table, table)


def test_layout_leaves_out_bad_requests() -> None:
    past, lens = np.array([3, -1, 0, 5, 0, 100]), np.array([4, 5, -2, 6, 7, 93])
    rows = np.array([0, 1, 2, 9, 3, 4])
    table = np.full((5, 12), 99, np.int32)
    out, got = run_layout(past, lens, table, rows, np.arange(20, dtype=np.int32), 16, 40, 4)
    keep = [0, 4]
    assert out.counts.tolist() == [11, 2, 1, kv8.LAYOUT_BAD_REQUEST]
    assert out.cu_q.tolist() == [0, 4, 4, 4, 4, 11, 11]
    assert out.positions.tolist()[:11] == [3, 4, 5, 6, 0, 1, 2, 3, 4, 5, 6]
    assert out.rows.tolist()[:11] == [99 * 16 + i for i in range(3, 7)] + list(range(7))
    assert sorted(out.tile_seq.tolist()) == [-1, -1] + keep
    assert got[3, 0] == 0 and (got[[0, 1, 2, 4]] == 99).all()


# -- the operators together ----------------------------------------------------------------------------------------


def test_layout_write_prefill_and_decode_together() -> None:
    """Two requests through a prompt in two chunks and a few decode steps, block tables built on the device."""
    rng = np.random.default_rng(51)
    heads, kv, dim, block, blocks = 4, 2, 64, 32, 30
    pool = kv8.Kv8Pool.allocate(1, blocks, block, kv, dim, DEV)
    cache = oracle.Cache(np.zeros((1, 2, blocks * 2, kv, 16, dim)), np.full((1, 2, blocks * 2, kv), -127))
    table = torch.full((2, 12), -1, dtype=torch.int32, device=DEV)
    free = dev(rng.permutation(blocks).astype(np.int32))
    cos, sin = helpers.rope_tables(dim, 400)
    past = np.zeros(2, np.int32)
    ws = torch.empty(kv8.decode_workspace_bytes(2, heads, kv, dim, 400), dtype=torch.uint8, device=DEV)
    for lens in ([150, 37], [20, 90], [1, 1], [1, 1], [1, 1]):
        total = sum(lens)
        decode = lens == [1, 1]
        plan = kv8.BatchLayout.allocate(2, total, 4, DEV)
        kv8.batch_layout_raw(dev(past), dev(lens, torch.int32), table, None, free, block, plan)
        counts = plan.counts.tolist()
        assert counts[0] == total and counts[3] == 0
        free = free[counts[2]:]
        q, k, v = (helpers.values(rng, "bf16", total, n, dim).to(DEV) for n in (heads, kv, kv))
        pos = plan.positions.cpu().numpy()
        slot = plan.rows.cpu().numpy()
        k_rot = oracle.rotate(f32(k), None, cos, sin, pos, 1)
        cache.write(0, slot, k_rot, f32(v))
        if decode:
            out = kv8.decode_attention_raw(q, k, v, pool, None, 0, table, None, plan.positions, dev(cos), dev(sin), 1,
                                           None,
                                           None, torch.empty_like(q), ws, 0.125)
            turned = oracle.rotate(f32(q), None, cos, sin, pos, 1).astype(np.float64)
        else:
            q_rot = torch.empty_like(q)
            kv8.write_raw(q, k, v, q_rot, pool, 0, plan.rows, plan.positions, dev(cos), dev(sin), 1, None, None)
            out = kv8.prefill_attention_raw(q_rot, pool, 0, table, dev([0, 1], torch.int32), plan.cu_q, dev(past),
                                            plan.tile_seq, plan.tile_q0, torch.empty_like(q), 0.125)
            turned = q_rot.cpu().double().numpy()
        helpers.same_cache(pool, cache)
        host = table.cpu().numpy()
        at = 0
        for s, n in enumerate(lens):
            seen = helpers.slots(host[s], np.arange(past[s] + n), block)
            want, bound = oracle.attend(turned[at:at + n], cache.values(0, 0, seen), cache.values(0, 1, seen),
                                        past[s] + np.arange(n), 0.125,
                                        **bounds("decode" if decode else "prefill", "bf16", dim, int(past[s] + n)))
            helpers.close(out[at:at + n], want, bound)
            at += n
        past = past + np.array(lens, np.int32)


def test_two_captured_decodes_share_a_workspace() -> None:
    """Graphs of different batches replayed in turn over one workspace, with an eager call between them."""
    cases = [DecodeCase(61, "bf16", 4, 2, 128, 1, False, 16, [2100, 5, 1300]),
             DecodeCase(62, "bf16", 4, 2, 128, 1, False, 16, [1025, 3000, 1024, 0, 2048])]
    ws = torch.full((max(c.workspace.nbytes for c in cases),), 255, dtype=torch.uint8, device=DEV)
    args = [c.args(ws=ws) for c in cases]
    want = [kv8.decode_attention_raw(*a.values()).clone() for a in args]  # appends; the same again changes nothing
    graphs = []
    for a in args:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            kv8.decode_attention_raw(*a.values())
    for turn in (0, 1, 0, 0, 1, 1, 0):
        args[turn]["out"].fill_(3.0)
        graphs[turn].replay()
        assert torch.equal(args[turn]["out"], want[turn])
        assert torch.equal(cases[1 - turn].run(ws=ws), want[1 - turn])


def test_layout_write_and_prefill_captured_together() -> None:
    """One graph lays out, writes and attends batches of other lengths than those it was captured with, padded to
    its capacity; what lies behind the last token stays as it was."""
    rng = np.random.default_rng(63)
    heads, kv, dim, block, blocks, tokens, tiles = 4, 2, 128, 16, 400, 500, 8
    pools = [kv8.Kv8Pool.allocate(2, blocks, block, kv, dim, DEV) for _ in range(2)]
    seed = torch.from_numpy(rng.integers(0, 120, size=pools[0].codes.shape).astype(np.uint8)).to(DEV)
    for p in pools:
        p.codes.view(torch.uint8).copy_(seed)
        p.scales.fill_(120)
    cos, sin = (dev(x) for x in helpers.rope_tables(dim, 2000))
    q, k, v = (helpers.values(rng, "bf16", tokens, n, dim).to(DEV) for n in (heads, kv, kv))
    fixed = rng.permutation(blocks).astype(np.int32)
    past, lens = dev([0, 0, 0], torch.int32), dev([1, 1, 1], torch.int32)
    free = dev(fixed[300:])
    start = np.full((3, 125), -1, np.int32)
    start[:, :100] = fixed[:300].reshape(3, 100)
    ws = torch.empty(kv8.prefill_workspace_bytes(tiles, 3, heads, dim), dtype=torch.uint8, device=DEV)

    def step(pool, table, plan, q_rot, out):
        kv8.batch_layout_raw(past, lens, table, None, free, block, plan)
        kv8.write_raw(q, k, v, q_rot, pool, 1, plan.rows, plan.positions, cos, sin, 1, None, None)
        kv8.prefill_attention_raw(q_rot, pool, 1, table, dev_rows, plan.cu_q, past, plan.tile_seq, plan.tile_q0, out,
                                  0.09, 3, ws)

    dev_rows = dev([0, 1, 2], torch.int32)
    sides = [(p, dev(start), kv8.BatchLayout.allocate(3, tokens, tiles, DEV), torch.empty_like(q), torch.empty_like(q))
             for p in pools]
    step(*sides[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*sides[0])
    pools[0].codes.view(torch.uint8).copy_(seed)
    pools[0].scales.fill_(120)
    for p, n in (([0, 1500, 31], [300, 1, 130]), ([16, 0, 1599], [0, 257, 200]), ([700, 700, 700], [0, 0, 0])):
        past.copy_(dev(p, torch.int32))
        lens.copy_(dev(n, torch.int32))
        for side in sides:
            side[1].copy_(dev(start))
            side[3].fill_(5.0)
            side[4].fill_(5.0)
        graph.replay()
        step(*sides[1])
        torch.cuda.synchronize()
        total = sum(n)
        for a, b in zip(*sides):
            if isinstance(a, torch.Tensor):
                assert torch.equal(a, b)
        for name in ("cu_q", "positions", "rows", "tile_seq", "tile_q0", "counts"):
            assert torch.equal(getattr(sides[0][2], name), getattr(sides[1][2], name))
        assert sides[0][2].counts.tolist()[0] == total and sides[0][2].counts.tolist()[3] == 0
        assert torch.equal(pools[0].codes.view(torch.uint8), pools[1].codes.view(torch.uint8))
        assert torch.equal(pools[0].scales, pools[1].scales)
        for t in sides[0][3:]:
            assert (t[total:] == 5.0).all() and torch.isfinite(t[:total]).all()


def test_blocks_past_4_gib_give_the_same_bits() -> None:
    """Write, prefill and decode through blocks whose codes lie past 2^32 bytes, against the same in a small pool."""
    rng = np.random.default_rng(64)
    heads, kv, dim, block, few, many = 16, 16, 128, 16, 130, 70_000
    lens, width = [1100, 700], 70
    assert (2 * many - 1) * kv * 16 * dim > 2 ** 32
    small = rng.permutation(few)[:sum(-(-(n + 1) // block) for n in lens)]
    q, k, v = (helpers.values(rng, "bf16", sum(lens) + 2, n, dim).to(DEV) for n in (heads, kv, kv))
    cos, sin = (dev(x) for x in helpers.rope_tables(dim, 1200))
    results = []
    for blocks, ids in ((few, small), (many, many - 1 - small)):
        pool = kv8.Kv8Pool.allocate(1, blocks, block, kv, dim, DEV)
        table = np.full((2, width), -1, np.int32)
        table[0, :69], table[1, :44] = ids[:69], ids[69:113]
        pos = np.concatenate([np.arange(n) for n in lens])
        rows = np.concatenate([helpers.slots(table[s], np.arange(n), block) for s, n in enumerate(lens)])
        q_rot, out = torch.empty_like(q[:-2]), torch.empty_like(q[:-2])
        kv8.write_raw(q[:-2], k[:-2], v[:-2], q_rot, pool, 0, dev(rows, torch.int64), dev(pos, torch.int32), cos, sin,
                      1, None, None)
        seq, q0 = ops.prefill_tiles(np.array(lens), np.zeros(2, np.int64))
        kv8.prefill_attention_raw(q_rot, pool, 0, dev(table), dev([0, 1], torch.int32),
                                  dev([0, lens[0], sum(lens)], torch.int32), dev([0, 0], torch.int32), dev(seq),
                                  dev(q0), out, 0.09)
        ws = torch.empty(kv8.decode_workspace_bytes(2, heads, kv, dim, 1200), dtype=torch.uint8, device=DEV)
        step = kv8.decode_attention_raw(q[-2:], k[-2:], v[-2:], pool, None, 0, dev(table), None, dev(lens, torch.int32),
                                        cos, sin, 1, None, None, torch.empty_like(q[-2:]), ws, 0.09)
        at = torch.from_numpy(ids.astype(np.int64)).to(DEV)
        results.append((out, step, pool.codes.view(torch.uint8)[:, :, at], pool.scales[:, :, at]))
        del pool
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert torch.isfinite(results[0][0]).all() and torch.isfinite(results[0][1]).all()


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("how", ["slot", "position", "padding"])
@pytest.mark.parametrize("dtype,heads,kv,dim,style,block", [("bf16", 3, 3, 128, 1, 16), ("f32", 2, 1, 96, 2, 32),
                                                            ("bf16", 2, 2, 64, 0, 16)])
def test_write_leaves_tokens_out_inside_a_tile(dtype, heads, kv, dim, style, block, how, many) -> None:
    """Tokens left out between others of their tile, in batches of which a wave takes one token or sixteen: the others
    are coded as one run, and the codes at their places stay as they were."""
    if how == "position" and style == 0:
        how = "slot"
    seqs = [(0, 40), (5, 30), (9, 3), (14, 20), (0, 16), (2, 13)] + ([(3, 1200), (0, 77)] if many else [])
    c = WriteCase(65, dtype, heads, kv, dim, style, False, block, seqs)
    rng = np.random.default_rng(66)
    out = rng.random(c.rows.size) < 0.3
    start = np.cumsum([0] + [n for _, n in seqs])
    out[start[0]:start[0] + 16] = [False] + [True] * 14 + [False]      # a tile's first and last token alone
    out[start[4]:start[4] + 16] = [True] * 3 + [False] + [True] * 11 + [False]  # not its first
    rows, pos = c.rows.copy(), c.pos.copy()
    if how == "padding":
        rows[out] = -1
    elif how == "slot":
        rows[out] = c.pool.num_blocks * block + c.rows[out]
    else:
        pos[out] = np.where(rng.random(out.sum()) < 0.5, -1, c.pos.max() + 1)
    got = c.run(rows=dev(rows), pos=dev(pos, torch.int32)).cpu()
    c.rows[out] = -1
    want = c.expect()
    left = torch.from_numpy(out)
    assert torch.equal(got[~left], want[~left])
    if how == "padding":
        assert (got[left] == 7.0).all()
    elif how == "position":
        assert got[left].isnan().all()
    else:
        assert torch.equal(got[left], want[left])
    helpers.same_cache(c.pool, c.cache)


@pytest.mark.parametrize("dtype,heads,kv", [("bf16", 4, 2), ("f32", 2, 1)])
def test_decode_rows_keep_their_bits_over_a_workspace_that_is_large_enough(dtype, heads, kv) -> None:
    """One workspace, sized for all rows and the longest context, past 64 chunks too: rows alone, in any order and in
    any company give the same bits."""
    contexts = [70_000, 5000, 1025, 3, 0, 2048, 66_000]
    c = DecodeCase(67, dtype, heads, kv, 64, 1, False, 64, contexts, layers=1)
    whole = c.run()
    for rows in ([0], [1], [6, 0], [2, 1, 5], [5, 4, 3, 2, 1]):
        r = torch.tensor(rows, device=DEV)
        a = c.args()
        part = c.run(q=c.q[r], k=c.k[r], v=c.v[r], layer=a["layer"][r], table=a["table"][r], pos=a["pos"][r],
                     out=torch.empty_like(whole[r]))
        assert torch.equal(part, whole[r])


def test_prefill_sequences_keep_their_bits_in_any_batch() -> None:
    """With the same number of parts."""
    c = PrefillCase(68, "bf16", 4, 2, 128, 16, [(700, 60), (0, 200), (300, 1), (1500, 129)])
    for splits in (1, 5):
        whole = c.run(splits=splits)
        for s in range(4):
            mine = slice(c.cu[s], c.cu[s + 1])
            seq, q0 = ops.prefill_tiles(c.new[s:s + 1], c.past[s:s + 1])
            ws = torch.empty(kv8.prefill_workspace_bytes(len(seq), splits, 4, 128), dtype=torch.uint8, device=DEV)
            part = kv8.prefill_attention_raw(c.q[mine], c.pool, c.layer, dev(c.table[s:s + 1]), dev([0], torch.int32),
                                             dev([0, int(c.new[s])], torch.int32), dev(c.past[s:s + 1], torch.int32),
                                             dev(seq), dev(q0), torch.empty_like(c.q[mine]), c.scale, splits, ws)
            assert torch.equal(part, whole[mine])


@pytest.mark.parametrize("dtype,heads,kv,dim", [("bf16", 4, 2, 128), ("f32", 2, 2, 64)])
def test_decode_rewrites_a_position_at_each_loop_step(dtype, heads, kv, dim) -> None:
    """The same positions again with other keys and values, smaller and larger ones, as a looped model that keeps one
    slot a position does: a tile keeps the larger scale, and starts anew at its first token."""
    c = DecodeCase(69, dtype, heads, kv, dim, 1, False, 16, [1, 2, 16, 17, 40, 300, 0, 1030], nan=True)
    rng = np.random.default_rng(70)
    for std in (1.0, 0.05, 3.0, 0.3):
        for t in (c.q, c.k, c.v):
            t.copy_(helpers.values(rng, dtype, *t.shape, std=1.0 if t is c.q else std))
        c.check()


@pytest.mark.parametrize("dtype,heads,kv,dim", [("bf16", 4, 2, 64), ("f32", 2, 2, 96), ("bf16", 2, 1, 128)])
@pytest.mark.parametrize("std,q_std", [(3.0, 1.5), (30.0, 0.05), (300.0, 0.006), (1e-4, 1.5)])
def test_decode_peaked_scores_and_growing_scales(dtype, heads, kv, dim, std, q_std) -> None:
    """New tokens that dwarf their tile's scale or vanish beside it, with queries of a size at which scores peak and a
    computation's error stays small: the bound is at most a quarter of each result."""
    c = DecodeCase(71, dtype, heads, kv, dim, 1, False, 16, [1, 2, 5, 16, 17, 18, 31, 270, 272, 273, 1500], std=std)
    c.q.copy_(helpers.values(np.random.default_rng(72), dtype, *c.q.shape, std=q_std))
    want, bound = c.expect()
    assert (np.linalg.norm(bound, axis=-1) < np.linalg.norm(want, axis=-1) / 4).all()
    helpers.close(c.run(), want, bound)
    helpers.same_cache(c.pool, c.cache)
