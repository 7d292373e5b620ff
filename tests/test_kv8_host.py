"""The 8-bit KV cache without a device: layout and oracle, sizes, and what the calls refuse."""

from __future__ import annotations

import copy
import ctypes
import dataclasses
import io

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import continuous_depth_batching_amd.ops  # noqa: F401  (registers the operators)
from continuous_depth_batching_amd import _lib, kv8
from oracle import kv8 as oracle
from tests import kv8_helpers as helpers

OPERATORS = {
    "kv8_write": {"codes", "scales"},
    "kv8_decode_attention": {"codes", "scales", "workspace"},
    "kv8_prefill_attention": {"workspace"},
    "batch_layout": {"block_table"},
}


@pytest.mark.parametrize("name", sorted(OPERATORS))
def test_operator_is_registered_with_its_mutations(name: str) -> None:
    op = getattr(torch.ops.cdb, name).default
    written = {a.name for a in op._schema.arguments if a.alias_info is not None and a.alias_info.is_write}
    assert written == OPERATORS[name]


def test_fake_implementations_give_output_shapes() -> None:
    with FakeTensorMode():
        def i32(*n):
            return torch.empty(n, dtype=torch.int32, device="cuda")

        q = torch.empty(40, 4, 64, dtype=torch.bfloat16, device="cuda")
        k = torch.empty(40, 2, 64, dtype=torch.bfloat16, device="cuda")
        codes = torch.empty(3, 2, 9, 2, 2, 1024, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        scales = torch.empty(3, 2, 9, 2, 2, dtype=torch.uint8, device="cuda")
        rows = torch.empty(40, dtype=torch.int64, device="cuda")
        cos = torch.empty(128, 32, device="cuda")
        ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
        out = torch.ops.cdb.kv8_write(q, k, k, codes, scales, 1, rows, i32(40), cos, cos, 1, None, None)
        assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
        out = torch.ops.cdb.kv8_decode_attention(q, k, k, codes, scales, None, 1, i32(40, 8), None, i32(40), cos, cos,
                                                 1, None, None, ws, 0.125)
        assert out.shape == q.shape and out.dtype == q.dtype
        out = torch.ops.cdb.kv8_prefill_attention(q, codes, scales, 1, i32(2, 8), i32(2), i32(3), i32(2), i32(2),
                                                  i32(2), 0.125, 1, None)
        assert out.shape == q.shape
        got = torch.ops.cdb.batch_layout(i32(5), i32(5), i32(5, 9), None, i32(7), 16, 100, 9)
        assert [tuple(x.shape) for x in got] == [(6,), (100,), (100,), (9,), (9,), (4,)]
        assert got[2].dtype == torch.int64


# -- the oracle against torch and closed forms --------------------------------------------------------------------


def test_oracle_rounds_as_the_type_does() -> None:
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy().astype(np.float64)
    finite = np.sort(np.unique(every[np.isfinite(every)]))
    mids = (finite[1:] + finite[:-1]) / 2
    x = np.concatenate([finite, mids, np.nextafter(mids, np.inf), np.nextafter(mids, -np.inf), [np.nan, np.inf]])
    got = oracle.round_e4m3(x)
    # In 64 bits torch's conversion sees a value that fp32 would have moved onto the tie; mids are exact in fp32.
    keep = x.astype(np.float32).astype(np.float64) == x
    want = torch.from_numpy(x[keep]).float().to(torch.float8_e4m3fn).float().numpy()
    np.testing.assert_array_equal(got[keep], want)
    up = np.nextafter(mids, np.inf)
    np.testing.assert_array_equal(oracle.round_e4m3(up), finite[1:])
    assert np.isnan(oracle.round_e4m3(np.array([np.inf]))).all()


@pytest.mark.parametrize("top,exponent", [(448.0, 0), (448.0001, 1), (1.75, -8), (1.76, -7), (0.0, -126),
                                          (2.0 ** -149, -126), (3.3e38, 120)])
def test_oracle_exponent(top: float, exponent: int) -> None:
    got = oracle.tile_exponent(np.array([0.0, -top, np.nan, np.inf]))
    assert got == exponent
    assert top <= 448 * 2.0 ** got and (got == -126 or top > 448 * 2.0 ** (got - 1))


def test_layout_round_trip() -> None:
    rng = np.random.default_rng(0)
    for dim, block in ((64, 16), (96, 32), (128, 64)):
        pool, cache = helpers.random_pool(rng, 2, 3, block, 5, dim, "cpu")
        helpers.same_cache(pool, cache)
        assert (pool.head_dim, pool.block_size, pool.num_kv_heads, pool.num_blocks) == (dim, block, 5, 3)
        k, v = pool.dequantize(1, torch.tensor([2, 0]))
        at = np.concatenate([np.arange(2 * block, 3 * block), np.arange(block)])
        np.testing.assert_array_equal(k.numpy(), cache.values(1, 0, at))
        np.testing.assert_array_equal(v.numpy(), cache.values(1, 1, at))


def test_oracle_attention_of_one_key_and_of_equal_keys() -> None:
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal((4, 2, 8)) for _ in range(3))
    out, bound = oracle.attend(q[:1], k, v, np.array([0]), 0.3, 2.0 ** -8, 0.0, 0.0)
    np.testing.assert_allclose(out[0], v[0])
    assert (bound <= 2.0 ** -8 * np.abs(v[0]) * 1.0001).all()
    out, _ = oracle.attend(q[:1], np.repeat(k[:1], 4, 0), v, np.array([3]), 0.3, 0.0, 0.0, 0.0)
    np.testing.assert_allclose(out[0], v.mean(0))


# -- sizes ---------------------------------------------------------------------------------------------------------


def test_workspace_sizes() -> None:
    assert kv8.decode_workspace_bytes(3, 8, 2, 128, 1025) >= 3 * 8 * 2 * 130 * 4
    assert kv8.decode_workspace_bytes(3, 8, 2, 128, 1024) < kv8.decode_workspace_bytes(3, 8, 2, 128, 1025)
    for bad in ((-1, 8, 2, 128, 1), (1, 0, 2, 128, 1), (1, 8, 2, 128, 0)):
        with pytest.raises(ValueError):
            kv8.decode_workspace_bytes(*bad)
    assert kv8.prefill_workspace_bytes(5, 1, 8, 128) == 0
    assert kv8.prefill_workspace_bytes(5, 3, 8, 128) >= 5 * 3 * 8 * 128 * 130 * 4
    with pytest.raises(ValueError):
        kv8.prefill_workspace_bytes(5, 0, 8, 128)


def test_prefill_splits_fill_the_device_and_keep_parts_long() -> None:
    assert kv8.prefill_splits(100, 16, 16, 1300) == 1      # a batch of fresh prompts fills it
    assert kv8.prefill_splits(4, 16, 16, 16128) > 1        # four chunks after long histories do not
    assert kv8.prefill_splits(1, 8, 1, 100) == 1           # too short to cut
    assert kv8.prefill_splits(0, 8, 1, 0) >= 1


# -- refusals ------------------------------------------------------------------------------------------------------

FAKE = ctypes.c_void_p(0x1000)  # every case is rejected on the host, before any device work
BF16 = _lib.CDB_DTYPE_BF16


@pytest.fixture(autouse=True)
def _no_device(request: pytest.FixtureRequest) -> None:
    if "without_gpu" in request.node.name and torch.cuda.is_available():
        pytest.skip("runs only where no device exists: the stand-in addresses must never reach a kernel")


def _write(**over):
    args = dict(q=FAKE, k=FAKE, v=FAKE, q_out=FAKE, codes=FAKE, scales=FAKE, layers=2, blocks=9, layer=1, rows=FAKE,
                positions=FAKE, cos=FAKE, sin=FAKE, style=1, max_positions=64, q_bias=None, k_bias=None, tokens=5,
                heads=8, kv=2, dim=128, block=16, q_stride=0, kv_stride=0, dtype=BF16, stream=None)
    args.update(over)
    return _lib.lib().cdb_kv8_write(*args.values())


@pytest.mark.parametrize("over,code", [
    (dict(k=None), "NULL"), (dict(v=None), "NULL"), (dict(rows=None), "NULL"), (dict(q=None), "NULL"),
    (dict(q_out=None), "NULL"), (dict(codes=None), "NULL"), (dict(scales=None), "NULL"), (dict(cos=None), "NULL"),
    (dict(positions=None), "NULL"), (dict(tokens=-1), "SHAPE"), (dict(layer=2), "SHAPE"), (dict(layer=-1), "SHAPE"),
    (dict(style=3), "UNSUPPORTED"), (dict(dim=80), "UNSUPPORTED"), (dict(dtype=7), "UNSUPPORTED"),
    (dict(block=8), "SHAPE"), (dict(block=48), "SHAPE"), (dict(blocks=0), "SHAPE"), (dict(kv=0), "SHAPE"),
    (dict(max_positions=0), "SHAPE"), (dict(q_stride=1023), "SHAPE"), (dict(kv_stride=255), "SHAPE"),
    (dict(codes=ctypes.c_void_p(0x1008)), "SHAPE"), (dict(q_out=ctypes.c_void_p(0x1002)), "SHAPE"),
    (dict(blocks=1 << 31), "SHAPE"), (dict(tokens=1 << 40), "SHAPE"),
])
def test_write_refusals_without_gpu(over, code) -> None:
    assert _write(**over) == getattr(_lib, "CDB_ERR_" + code)


def _decode(**over):
    args = dict(q=FAKE, k=FAKE, v=FAKE, codes=FAKE, scales=FAKE, layers=2, blocks=9, cache_layer=None, cache_layer0=0,
                table=FAKE, table_row=None, table_rows=4, table_width=8, seqlens=FAKE, cos=FAKE, sin=FAKE, style=1,
                max_positions=64, q_bias=None, k_bias=None, out=FAKE, workspace=FAKE, workspace_bytes=1 << 20, rows=4,
                heads=8, kv=2, dim=128, block=16, scale=0.1, q_stride=0, kv_stride=0, dtype=BF16, stream=None)
    args.update(over)
    return _lib.lib().cdb_kv8_decode_attention(*args.values())


@pytest.mark.parametrize("over,code", [
    (dict(q=None), "NULL"), (dict(k=None), "NULL"), (dict(v=None), "NULL"), (dict(codes=None), "NULL"),
    (dict(table=None), "NULL"), (dict(seqlens=None), "NULL"), (dict(out=None), "NULL"), (dict(workspace=None), "NULL"),
    (dict(sin=None), "NULL"), (dict(heads=7), "SHAPE"), (dict(heads=0), "SHAPE"), (dict(rows=-1), "SHAPE"),
    (dict(rows=5), "SHAPE"), (dict(table_width=0), "SHAPE"), (dict(table_width=1 << 27), "SHAPE"),
    (dict(dim=32), "UNSUPPORTED"), (dict(block=24), "SHAPE"), (dict(dtype=2), "UNSUPPORTED"),
    (dict(style=-1), "UNSUPPORTED"), (dict(scale=0.0), "SHAPE"), (dict(scale=float("nan")), "SHAPE"),
    (dict(scale=float("inf")), "SHAPE"), (dict(workspace_bytes=4 * 8 * 130 * 4 - 1), "CAPACITY"),
    (dict(workspace_bytes=-1), "CAPACITY"), (dict(workspace=ctypes.c_void_p(0x1004)), "SHAPE"),
    (dict(q_stride=8), "SHAPE"), (dict(kv_stride=8), "SHAPE"), (dict(max_positions=0), "SHAPE"),
])
def test_decode_refusals_without_gpu(over, code) -> None:
    assert _decode(**over) == getattr(_lib, "CDB_ERR_" + code)


def _prefill(**over):
    args = dict(q=FAKE, codes=FAKE, scales=FAKE, layers=2, blocks=9, layer=0, table=FAKE, table_row=FAKE, table_rows=4,
                table_width=8, cu=FAKE, past=FAKE, seqs=2, tile_seq=FAKE, tile_q0=FAKE, tiles=3, out=FAKE, tokens=300,
                splits=1, workspace=None, workspace_bytes=0, heads=8, kv=2, dim=128, block=16, scale=0.1, dtype=BF16,
                stream=None)
    args.update(over)
    return _lib.lib().cdb_kv8_prefill_attention(*args.values())


@pytest.mark.parametrize("over,code", [
    (dict(q=None), "NULL"), (dict(out=None), "NULL"), (dict(codes=None), "NULL"), (dict(table=None), "NULL"),
    (dict(table_row=None), "NULL"), (dict(cu=None), "NULL"), (dict(past=None), "NULL"), (dict(tile_seq=None), "NULL"),
    (dict(splits=2), "NULL"), (dict(splits=0), "SHAPE"), (dict(splits=70000), "SHAPE"),
    (dict(splits=2, workspace=FAKE, workspace_bytes=100), "CAPACITY"), (dict(layer=2), "SHAPE"),
    (dict(heads=9), "SHAPE"), (dict(tokens=-1), "SHAPE"), (dict(tiles=-1), "SHAPE"), (dict(seqs=-1), "SHAPE"),
    (dict(table_width=0), "SHAPE"), (dict(dim=256), "UNSUPPORTED"), (dict(block=0), "SHAPE"),
    (dict(scale=-1.0), "SHAPE"), (dict(q=ctypes.c_void_p(0x1008)), "SHAPE"), (dict(dtype=-1), "UNSUPPORTED"),
])
def test_prefill_refusals_without_gpu(over, code) -> None:
    assert _prefill(**over) == getattr(_lib, "CDB_ERR_" + code)


def _layout(**over):
    args = dict(past=FAKE, lens=FAKE, seqs=3, table=FAKE, table_row=None, table_rows=4, table_width=8, free=FAKE,
                num_free=9, block=16, cu=FAKE, positions=FAKE, rows=FAKE, tokens=64, tile_seq=FAKE, tile_q0=FAKE,
                tiles=8, counts=FAKE, stream=None)
    args.update(over)
    return _lib.lib().cdb_batch_layout(*args.values())


@pytest.mark.parametrize("over,code", [
    (dict(past=None), "NULL"), (dict(lens=None), "NULL"), (dict(table=None), "NULL"), (dict(free=None), "NULL"),
    (dict(cu=None), "NULL"), (dict(positions=None), "NULL"), (dict(rows=None), "NULL"), (dict(tile_q0=None), "NULL"),
    (dict(counts=None), "NULL"), (dict(seqs=-1), "SHAPE"), (dict(seqs=4001), "SHAPE"), (dict(seqs=5), "SHAPE"),
    (dict(table_width=0), "SHAPE"), (dict(block=12), "SHAPE"), (dict(block=0), "SHAPE"), (dict(tokens=-1), "SHAPE"),
    (dict(tiles=-1), "SHAPE"), (dict(num_free=-1), "SHAPE"), (dict(table_width=1 << 27), "SHAPE"),
])
def test_layout_refusals_without_gpu(over, code) -> None:
    assert _layout(**over) == getattr(_lib, "CDB_ERR_" + code)


def test_nothing_to_do_is_no_error_without_gpu() -> None:
    assert _write(tokens=0) == _lib.CDB_OK
    assert _decode(rows=0) == _lib.CDB_OK
    assert _prefill(tiles=0) == _lib.CDB_OK and _prefill(seqs=0) == _lib.CDB_OK and _prefill(tokens=0) == _lib.CDB_OK


def test_pool_refusals() -> None:
    for block in (8, 24, 0):
        with pytest.raises(ValueError):
            kv8.Kv8Pool.allocate(1, 2, block, 2, 64, "cpu")
    pool = kv8.Kv8Pool.allocate(1, 2, 32, 2, 64, "cpu")
    with pytest.raises(TypeError):
        kv8.Kv8Pool(pool.codes.view(torch.uint8), pool.scales)
    with pytest.raises(ValueError):
        kv8.Kv8Pool(pool.codes, pool.scales[:, :, :1])
    with pytest.raises(ValueError):
        kv8.Kv8Pool(pool.codes[:, :, :, :1], pool.scales[:, :, :, :1])


def _python_args():
    pool = kv8.Kv8Pool.allocate(1, 4, 16, 2, 64, "cpu")
    q, k = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64)
    rows, pos = torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int32)
    cos = torch.zeros(8, 32)
    return pool, q, k, rows, pos, cos


def test_python_write_checks() -> None:
    pool, q, k, rows, pos, cos = _python_args()

    def call(q=q, k=k, v=k, q_out=q, layer=0, rows=rows, pos=pos, cos=cos, style=1, qb=None, kb=None):
        kv8.write_raw(q, k, v, q_out, pool, layer, rows, pos, cos, cos, style, qb, kb)

    with pytest.raises(RuntimeError, match="GPU only"):
        call()
    for bad in (dict(q=None), dict(q=q[:2]), dict(q_out=q[:, :2]), dict(k=k[:, :1]), dict(v=k.bfloat16()),
                dict(layer=1),
                dict(rows=rows[:2]), dict(cos=cos[:, :16]), dict(style=3), dict(qb=torch.zeros(4, 32)),
                dict(kb=torch.zeros(2, 64).bfloat16())):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(TypeError):
        call(rows=rows.int())
    wide = torch.zeros(3, 2, 128)[..., ::2]
    with pytest.raises((ValueError, RuntimeError)):
        call(k=wide, v=wide)


def test_python_decode_checks() -> None:
    pool, q, k, _, pos, cos = _python_args()
    table, ws = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(1 << 16, dtype=torch.uint8)

    def call(q=q, k=k, v=k, layer=None, table=table, trow=None, pos=pos, cos=cos, style=1, out=q, ws=ws):
        kv8.decode_attention_raw(q, k, v, pool, layer, 0, table, trow, pos, cos, cos, style, None, None, out, ws, 0.1)

    with pytest.raises(RuntimeError, match="GPU only"):
        call()
    for bad in (dict(q=torch.zeros(3, 3, 64), out=torch.zeros(3, 3, 64)), dict(k=k[:2]), dict(out=q[:2]),
                dict(table=table[:2]), dict(table=table[0]), dict(pos=pos[:2]), dict(trow=pos[:1]), dict(layer=pos[:1]),
                dict(cos=cos.double()), dict(q=torch.zeros(3, 0, 64), out=torch.zeros(3, 0, 64))):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(k=k.bfloat16(), v=k.bfloat16()), dict(pos=pos.long()), dict(table=table.long())):
        with pytest.raises(TypeError):
            call(**bad)


def test_python_prefill_and_layout_checks() -> None:
    pool, q, _, _, pos, _ = _python_args()
    table, cu, one = torch.zeros(1, 2, dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32), pos[:1]

    def call(q=q, layer=0, table=table, cu=cu, tiles=one, out=q, splits=1):
        kv8.prefill_attention_raw(q, pool, layer, table, one, cu, one, tiles, one, out, 0.1, splits)

    with pytest.raises(RuntimeError, match="GPU only"):
        call()
    for bad in (dict(q=q[:, :3], out=q[:, :3]), dict(layer=1), dict(table=table[0]), dict(cu=cu[:1]),
                dict(tiles=pos[:2]), dict(out=q[:2]), dict(splits=2)):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(TypeError):
        call(cu=cu.long())

    a = kv8.BatchLayout.allocate(3, 8, 4, "cpu")
    free = torch.zeros(4, dtype=torch.int32)
    tables = torch.zeros(3, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        kv8.batch_layout_raw(pos, pos, tables, None, free, 16, a)
    for args in ((pos, pos[:2], tables, None), (pos, pos, tables[:2], None), (pos, pos, tables[0], None),
                 (pos[:2], pos[:2], tables, None), (pos, pos, tables, pos[:2])):
        with pytest.raises(ValueError):
            kv8.batch_layout_raw(*args, free, 16, a)
    with pytest.raises(TypeError):
        kv8.batch_layout_raw(pos, pos, tables.long(), None, free, 16, a)


@pytest.mark.parametrize("seqs,tokens,tiles", [(3, 8, 4), (0, 0, 0), (1, 7, 1), (4000, 1, 0)])
def test_a_layouts_buffers_are_where_its_tensors_say(seqs, tokens, tiles) -> None:
    a = kv8.BatchLayout.allocate(seqs, tokens, tiles, "cpu")
    parts = (a.cu_q, a.positions, a.rows, a.tile_seq, a.tile_q0, a.counts)
    assert [t.numel() for t in parts] == [seqs + 1, tokens, tokens, tiles, tiles, 4]
    assert a.rows.dtype is torch.int64 and all(t.dtype is torch.int32 for t in parts if t is not a.rows)
    b = kv8.BatchLayout(*parts)
    assert a._num_seqs == b._num_seqs == seqs

    def pointers(x):  # an empty tensor's is null
        p = x._args
        return (p[0], p[1] if tokens else 0, p[2] if tokens else 0, p[3], p[4] if tiles else 0, p[5] if tiles else 0,
                p[6], p[7])

    assert pointers(a) == pointers(b)


def test_layout_refuses_buffers_that_do_not_fit() -> None:
    a = kv8.BatchLayout.allocate(3, 8, 4, "cpu")
    for bad in (dict(rows=a.positions), dict(positions=a.rows), dict(counts=a.counts.long())):
        with pytest.raises(TypeError):
            dataclasses.replace(a, **bad)
    wide = torch.zeros(16, dtype=torch.int32)
    for bad in (dict(rows=a.rows[:7]), dict(positions=a.positions[:7]), dict(tile_q0=a.tile_q0[:3]),
                dict(counts=a.counts[:3]), dict(positions=wide[::2]), dict(tile_seq=wide[::4]),
                dict(cu_q=torch.zeros(0, dtype=torch.int32)),
                dict(cu_q=torch.zeros(4, dtype=torch.int32, device="meta"))):
        with pytest.raises(ValueError):
            dataclasses.replace(a, **bad)
    with pytest.raises(ValueError, match="3 requests"):
        pos = torch.zeros(2, dtype=torch.int32)
        kv8.batch_layout_raw(pos, pos, torch.zeros(2, 2, dtype=torch.int32), None, pos, 16, a)


def test_oracle_codes_a_run_over_tokens_left_out() -> None:
    rng = np.random.default_rng(2)
    codes, exps = np.full((1, 2, 2, 1, 16, 4), 3.0), np.full((1, 2, 2, 1), -7)
    k = rng.standard_normal((6, 1, 4)).astype(np.float32) * np.float32(2.0) ** np.arange(6)[:, None, None]
    cache = oracle.Cache(codes.copy(), exps)
    cache.write(0, np.array([16 + 2, -1, 16 + 4, 16 + 5, -1, 0]), k, k)
    top = oracle.tile_exponent(k[[0, 2, 3]])
    assert (cache.exponents[0, :, 1, 0] == max(top, -7)).all()
    got = cache.codes[0, 0, 1, 0]
    for slot, t in ((2, 0), (4, 2), (5, 3)):
        np.testing.assert_array_equal(got[slot], oracle.round_e4m3(k[t, 0] * 2.0 ** -float(top)))
    assert (got[[3] + list(range(6, 16))] == 3.0).all() and (got[:2] == oracle.round_e4m3(3.0 * 2.0 ** (-7.0 - top))).all()
    assert cache.exponents[0, 0, 0, 0] == oracle.tile_exponent(k[5])


# -- a call reaches the memory that its tensors have when it is made ----------------------------------------------


class _Recorder:
    """Stands in for the library: keeps the last call's arguments and answers that all is well."""

    def __getattr__(self, name):
        def call(*args):
            self.name, self.args = name, args
            return 0
        return call


@pytest.fixture
def recorder(monkeypatch):
    r = _Recorder()
    monkeypatch.setattr(kv8._lib, "lib", lambda: r)
    monkeypatch.setattr(kv8, "_require_here", lambda *tensors: None)
    monkeypatch.setattr(kv8, "_stream", lambda: 0)
    return r


def _deep(x):
    return copy.deepcopy(x)


def _saved(x):
    buffer = io.BytesIO()
    torch.save(x, buffer)
    buffer.seek(0)
    return torch.load(buffer, weights_only=False)


def _moved(x):
    """The same object, its tensors moved to other storages in place."""
    for f in dataclasses.fields(x):
        t = getattr(x, f.name)
        t.data = t.detach().clone()
    return x


def _set(x):
    for f in dataclasses.fields(x):
        t = getattr(x, f.name)
        t.set_(t.detach().clone())
    return x


ANOTHER = [_deep, _saved, _moved, _set, copy.copy]


@pytest.mark.parametrize("another", ANOTHER)
def test_calls_on_another_pool_reach_its_own_memory(recorder, another) -> None:
    pool, q, k, rows, pos, cos = _python_args()
    pool = another(pool)
    own = (pool.codes.data_ptr(), pool.scales.data_ptr(), 1, 4)
    kv8.write_raw(q, k, k, q, pool, 0, rows, pos, cos, cos, 1, None, None)
    assert recorder.name == "cdb_kv8_write" and recorder.args[4:8] == own
    table, ws = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(1 << 16, dtype=torch.uint8)
    kv8.decode_attention_raw(q, k, k, pool, None, 0, table, None, pos, cos, cos, 1, None, None, q, ws, 0.1)
    assert recorder.name == "cdb_kv8_decode_attention" and recorder.args[3:7] == own
    cu, one = torch.tensor([0, 3], dtype=torch.int32), pos[:1]
    kv8.prefill_attention_raw(q, pool, 0, table, one, cu, one, one, one, q, 0.1)
    assert recorder.name == "cdb_kv8_prefill_attention" and recorder.args[1:5] == own


@pytest.mark.parametrize("made,another", [(m, a) for m in ("allocated", "given") for a in ANOTHER
                                          if (m, a) != ("allocated", _saved)])  # torch does not save such views
def test_calls_on_another_layout_reach_its_own_memory(recorder, another, made) -> None:
    a = kv8.BatchLayout.allocate(3, 8, 4, "cpu")
    if made == "given":
        a = kv8.BatchLayout(*(getattr(a, f.name).clone() for f in dataclasses.fields(a)))
    a = another(a)
    pos, free = torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    kv8.batch_layout_raw(pos, pos, torch.zeros(3, 2, dtype=torch.int32), None, free, 16, a)
    assert recorder.args[-9:-1] == (a.cu_q.data_ptr(), a.positions.data_ptr(), a.rows.data_ptr(), 8,
                                    a.tile_seq.data_ptr(), a.tile_q0.data_ptr(), 4, a.counts.data_ptr())


def test_buffers_changed_after_they_were_checked_are_checked_again(recorder) -> None:
    pool, q, k, rows, pos, cos = _python_args()
    pool.codes.resize_(1, 2, 9, 2, 1, 1024)
    with pytest.raises(ValueError, match="scales match"):
        kv8.write_raw(q, k, k, q, pool, 0, rows, pos, cos, cos, 1, None, None)
    free = torch.zeros(4, dtype=torch.int32)
    for change in (lambda a: a.positions.resize_(9), lambda a: a.tile_q0.resize_(3), lambda a: a.counts.resize_(3),
                   lambda a: a.cu_q.resize_(9), lambda a: a.rows.resize_(7)):
        a = kv8.BatchLayout(*(getattr(x, f.name).clone() for x in [kv8.BatchLayout.allocate(3, 8, 4, "cpu")]
                              for f in dataclasses.fields(x)))
        change(a)
        with pytest.raises(ValueError):
            kv8.batch_layout_raw(pos, pos, torch.zeros(3, 2, dtype=torch.int32), None, free, 16, a)


def _views(rows: int, heads: int, dim: int) -> dict[str, torch.Tensor]:
    """Views that no call can read by a row stride and dense heads, with a word of what is said of each."""

    whole = torch.zeros(rows, heads, 2 * dim)
    return {
        "contiguous heads": whole[..., ::2],
        "contiguous heads ": whole[..., :dim],
        "rows overlap": torch.zeros(1, heads, dim).expand(rows, heads, dim),
        "rows overlap ": torch.zeros((rows + 1) * heads * dim).as_strided((rows, heads, dim), (dim, dim, 1)),
    }


@pytest.mark.parametrize("which", ["q", "k", "v"])
@pytest.mark.parametrize("view", sorted(_views(3, 2, 64)))
def test_write_and_decode_refuse_views_they_cannot_read(which, view) -> None:
    pool, q, k, rows, pos, cos = _python_args()
    given = dict(q=q, k=k, v=k) | {which: _views(3, 4 if which == "q" else 2, 64)[view]}
    with pytest.raises(ValueError, match=view.strip()):
        kv8.write_raw(*given.values(), q, pool, 0, rows, pos, cos, cos, 1, None, None)
    table, ws = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(1 << 16, dtype=torch.uint8)
    with pytest.raises(ValueError, match=view.strip()):
        kv8.decode_attention_raw(*given.values(), pool, None, 0, table, None, pos, cos, cos, 1, None, None, q, ws, 0.1)


def test_write_and_decode_refuse_keys_and_values_of_different_strides() -> None:
    pool, q, k, rows, pos, cos = _python_args()
    wide = torch.zeros(3, 5, 64)[:, :2]
    for key, value in ((k, wide), (wide, k)):
        with pytest.raises(ValueError, match="stride"):
            kv8.write_raw(q, key, value, q, pool, 0, rows, pos, cos, cos, 1, None, None)
        table, ws = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(1 << 16, dtype=torch.uint8)
        with pytest.raises(ValueError, match="stride"):
            kv8.decode_attention_raw(q, key, value, pool, None, 0, table, None, pos, cos, cos, 1, None, None, q, ws,
                                     0.1)


def test_row_strides_that_calls_take() -> None:
    assert kv8._row_stride("x", torch.zeros(3, 5, 64)[:, 1:3], 3, 2, 64) == 5 * 64
    assert kv8._row_stride("x", torch.zeros(3, 2, 64), 3, 2, 64) == 2 * 64
    assert kv8._row_stride("x", torch.zeros(3, 9, 64)[:, ::9], 3, 1, 64) == 9 * 64      # one head: its stride is free
    assert kv8._row_stride("x", torch.zeros(1, 2, 64).expand(1, 2, 64), 1, 2, 64) == 2 * 64
