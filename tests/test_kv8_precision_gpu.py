"""The 8-bit attention kernels where single keys or tiles dwarf the rest, against the definition in 64 bits with
bounds that the small ones' share alone has to meet."""

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
KINDS = ["decode", "prefill", "split"]


def numerics(kind: str, dtype: str, dim: int, tokens: int) -> dict[str, float]:
    """What a computation rounds, relative (``expect``).

    Scores: dim products summed in fp32 for each part of the query, and a few roundings of scaling. A prefill query in
    bf16 is its own single part; fp32 queries are three bf16 parts (2^-24 left of each element); a bf16 decode query
    is 3 e4m3 parts, 2^-13.8 of the head's largest element, whose products keep some 2^-16 of their largest term.
    Probabilities: an fp16 part leaves 2^-12 of them (2^-11 is counted) and half of fp16's smallest step, 2^-25. They
    are raised by 2^15 in decode, whose largest probability is 1, and by 2^9 in prefill, where it may be 2^6. fp32
    models take what is left as a second part that is 2^11 larger: 2^-23, and the step 2^-11 of the first's. The
    exponential, its argument and the fp32 sums over tokens besides. The result: half a step of its type, divisions
    and joins."""
    wide = dtype == "f32"
    if kind == "decode":
        parts, left, top = (3, TINY, 0.0) if wide else (3, 0.0, 2.0 ** -13.8 + 3 * 2.0 ** -16)
    else:
        parts, left, top = (3, TINY, 0.0) if wide else (1, 0.0, 0.0)
    return dict(round_off=(16 * TINY if wide else 2.0 ** -8 + 8 * TINY), score_off=(parts * dim + 8) * TINY + left,
                top_off=top, prob_off=(2.0 ** -23 if wide else 2.0 ** -11) + (2 * tokens + 16) * TINY,
                floor=(2.0 ** -40 if kind == "decode" else 2.0 ** -34) * (2.0 ** -11 if wide else 1.0))


def expect(q, k, v, end, scale, round_off, score_off, top_off, prob_off, floor):
    """Attention of q [n, H, D] over k, v [tokens, Hkv, D] in 64 bits, query i over keys 0..end[i], and the bound of
    ``oracle.kv8.attend`` with each probability's floor counted for no more than the probability itself (a smaller
    one is at worst left out)."""
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    group = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        kh, vh = k[:, h // group], v[:, h // group]
        s = q[:, h] @ kh.T * scale
        size = np.abs(q[:, h])
        mass = (score_off * size + top_off * size.max(1, keepdims=True)) @ np.abs(kh).T * scale
        for i in range(len(q)):
            n = end[i] + 1
            p = np.exp(s[i, :n] - s[i, :n].max())
            p /= p.sum()
            a = np.abs(vh[:n])
            out[i, h] = p @ vh[:n]
            grown = (1 + round_off) * np.expm1(2 * mass[i, :n].max() + prob_off)
            bound[i, h] = round_off * np.abs(out[i, h]) + grown * (p @ a) + np.minimum(p, floor) @ a
    return out, bound


class Sequence:
    """One sequence of n tokens of a kind's call: a decode step's last token, or a prefill chunk of the last ``new``.
    ``keys`` and ``values`` [n, Hkv, D] are codes, ``k_exp`` and ``v_exp`` the exponents of its tiles."""

    def __init__(self, kind, dtype, heads, kv, dim, keys, values, k_exp, v_exp, q, new=40):
        n, tiles = keys.shape[0], -(-keys.shape[0] // 16)
        rng = np.random.default_rng(3)
        self.kind, self.dtype, self.dim, self.n = kind, dtype, dim, n
        self.new = 1 if kind == "decode" else new
        perm = rng.permutation(tiles + 1).astype(np.int32)
        self.table = perm[None, :tiles].copy()
        codes = np.zeros((1, 2, tiles + 1, kv, 16, dim))
        exps = np.full((1, 2, tiles + 1, kv), -6)
        at = helpers.slots(self.table[0], np.arange(n), 16)
        for plane, (c, e) in enumerate(((keys, k_exp), (values, v_exp))):
            codes[0, plane, at // 16, :, at % 16] = c
            exps[0, plane, self.table[0]] = e[:, None]
        self.cache = oracle.Cache(codes, exps)
        scales = torch.from_numpy((exps + 127).astype(np.uint8))[:, :, :, None].transpose(3, 4).contiguous()
        self.pool = kv8.Kv8Pool(helpers.pack(codes, 16).to(DEV), scales.to(DEV))
        self.q = torch.from_numpy(q).to(helpers.TYPES[dtype]).to(DEV)
        self.scale, self.at = dim ** -0.5, at

    def run(self, k_new=None, v_new=None):
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)
        out = torch.empty_like(self.q)
        heads, kv = self.q.shape[1], self.pool.num_kv_heads
        if self.kind == "decode":
            ws = torch.empty(kv8.decode_workspace_bytes(1, heads, kv, self.dim, self.n), dtype=torch.uint8, device=DEV)
            self.cache.append(0, int(self.at[-1]), k_new.float().cpu().numpy(), v_new.float().cpu().numpy())
            return kv8.decode_attention_raw(self.q, k_new, v_new, self.pool, None, 0, t(self.table), None,
                                            t([self.n - 1]), None, None, 0, None, None, out, ws, self.scale)
        past = self.n - self.new
        seq, q0 = ops.prefill_tiles(np.array([self.new]), np.array([past]))
        splits = 3 if self.kind == "split" else 1
        ws = torch.empty(kv8.prefill_workspace_bytes(len(seq), splits, heads, self.dim), dtype=torch.uint8, device=DEV)
        return kv8.prefill_attention_raw(self.q, self.pool, 0, t(self.table), t([0]), t([0, self.new]), t([past]),
                                         t(seq), t(q0), out, self.scale, splits, ws)

    def expect(self):
        k, v = (self.cache.values(0, plane, self.at) for plane in (0, 1))
        end = np.arange(self.n - self.new, self.n)
        return expect(self.q.double().cpu().numpy(), k, v, end, self.scale,
                      **numerics(self.kind, self.dtype, self.dim, self.n))

    def new_token(self, rng, key=0.0):
        """A decode step's key (all ``key`` in element 0) and value."""
        kv = self.pool.num_kv_heads
        k = torch.zeros(1, kv, self.dim)
        k[..., 0] = key
        v = helpers.values(rng, self.dtype, 1, kv, self.dim)
        return k.to(self.q.dtype).to(DEV), v.to(DEV)

    def check(self, rng, **token):
        got = self.run(*self.new_token(rng, **token)) if self.kind == "decode" else self.run()
        want, bound = self.expect()
        helpers.close(got, want, bound)
        # The bound says something: a result of zeros is four times past it. (Relative to sum(p |v|) it is some
        # 2^-8; values of random signs leave sum(p v) up to sqrt(tokens) = 39 times smaller than that.)
        assert (np.linalg.norm(bound, axis=-1) < np.linalg.norm(want, axis=-1) / 4).all()


def line(rng, n, kv, dim, first):
    """Codes of keys that score ``first`` (by their element 0 alone), and of values over most of their range."""
    keys = np.zeros((n, kv, dim))
    keys[:, :, 0] = oracle.round_e4m3(first)[:, None]
    return keys, oracle.round_e4m3(np.clip(rng.standard_normal((n, kv, dim)) * 90, -448, 448))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,heads,kv,dim", [("bf16", 4, 2, 128), ("f32", 2, 2, 64), ("f32", 2, 1, 128),
                                                ("bf16", 3, 3, 96), ("bf16", 2, 2, 64), ("f32", 1, 1, 96)])
def test_keys_far_below_a_sink_keep_their_share(kind, dtype, heads, kv, dim) -> None:
    """A first key that outscores all others by 2^27..2^21 and whose value is zero: what is left is theirs."""
    rng = np.random.default_rng(71)
    n = 1500
    keys, values = line(rng, n, kv, dim, np.concatenate([[448.0], rng.uniform(0.0, 96.0, n - 1)]))
    values[0] = 0.0
    tiles = -(-n // 16)
    k_exp, v_exp = np.full(tiles, -4), rng.integers(-7, -4, tiles)
    q = np.zeros((1 if kind == "decode" else 40, heads, dim))
    q[:, :, 0] = 27 * np.log(2.0) / 28 * dim ** 0.5  # the sink's key is 448 / 16
    Sequence(kind, dtype, heads, kv, dim, keys, values, k_exp, v_exp, q).check(rng)


def spread_values(rng, tiles, pattern, apart):
    """Exponents of the value tiles: ``pattern`` says which are 2^apart larger."""
    big = {"first": np.arange(tiles) < 2, "last": np.arange(tiles) >= tiles - 2, "middle": np.arange(tiles) == 50,
           "every other": np.arange(tiles) % 2 == 1, "every other pair": np.arange(tiles) // 2 % 2 == 0}[pattern]
    return big, np.where(big, apart - 5, rng.integers(-7, -4, tiles))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("apart", [14, 24, 55])
@pytest.mark.parametrize("pattern", ["first", "last", "middle", "every other", "every other pair"])
@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f32", 64), ("bf16", 96)])
def test_values_far_below_others_keep_their_share(kind, apart, pattern, dtype, dim) -> None:
    """Tiles of values 2^apart larger, that keys of next to no probability keep out of the result."""
    rng = np.random.default_rng(72)
    n = 1497
    tiles = -(-n // 16)
    big, v_exp = spread_values(rng, tiles, pattern, apart)
    far = np.repeat(big, 16)[:n]
    if kind == "decode":
        far[-1] = False  # the new token is one of the others, in a tile of large values or not
        if pattern == "last":
            v_exp[-1], big[-1] = -6, False
    # Scores: 0..2 in units of log2 for the small ones, -112 for the large ones (a code of -448 over a key's of 8).
    first = np.where(far, -448.0, rng.uniform(0.0, 8.0, n))
    keys, values = line(rng, n, 2, dim, first)
    values = np.abs(values)  # sums that do not cancel: the bound stays small beside them
    if kind != "decode" and big[-1]:
        keys[-40:, :, 0] = 0.0  # the queries' own tokens: see the next test
        far[-40:] = False
        v_exp[-3:] = -6
    q = np.zeros((1 if kind == "decode" else 40, 2, dim))
    q[:, :, 0] = 112 * np.log(2.0) / 28 * dim ** 0.5
    Sequence(kind, dtype, 2, 2, dim, keys, values, np.full(tiles, -4), v_exp, q).check(rng)


@pytest.mark.parametrize("kind", ["prefill", "split"])
@pytest.mark.parametrize("apart", [20, 50])
@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f32", 64), ("bf16", 96)])
def test_values_of_later_tokens_leave_earlier_queries_alone(kind, apart, dtype, dim) -> None:
    """A chunk whose every other tile holds values 2^apart larger: queries before the first of them see none."""
    rng = np.random.default_rng(73)
    n, new = 70, 70
    tiles = -(-n // 16)
    v_exp = np.where(np.arange(tiles) % 2 == 1, apart - 5, -5)
    keys = oracle.round_e4m3(np.clip(rng.standard_normal((n, 2, dim)) * 40, -448, 448))
    values = oracle.round_e4m3(np.clip(rng.standard_normal((n, 2, dim)) * 90, -448, 448))
    q = rng.standard_normal((new, 2, dim)) * 0.5
    s = Sequence(kind, dtype, 2, 2, dim, keys, values, np.full(tiles, -5), v_exp, q, new=new)
    got = s.run()
    want, bound = s.expect()
    helpers.close(got, want, bound)
    assert (np.linalg.norm(bound[:16], axis=-1) < np.linalg.norm(want[:16], axis=-1) / 4).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("f32", 128), ("bf16", 96)])
@pytest.mark.parametrize("plane,byte", [(0, 0), (0, 255), (1, 0), (1, 255)])
def test_scale_bytes_outside_their_range_are_read_as_its_ends(kind, dtype, dim, plane, byte) -> None:
    """0 as 1 and 255 as 254, by every call and by ``dequantize``, with queries that make such keys matter."""
    rng = np.random.default_rng(74)
    n, end = 300, -126 if byte == 0 else 127
    tiles = -(-n // 16)
    keys, values = line(rng, n, 2, dim, rng.uniform(0.0, 96.0, n))
    values = np.abs(values)
    k_exp, v_exp = np.full(tiles, -4), np.full(tiles, -6)
    (k_exp, v_exp)[plane][:] = end
    if byte == 255:  # within fp32: codes of up to 2^-6
        (keys, values)[plane][:] = oracle.round_e4m3((keys, values)[plane] * 2.0 ** -14)
    unit = np.abs(keys).max() * 2.0 ** float(k_exp[0])
    q = np.zeros((1 if kind == "decode" else 40, 2, dim))
    q[:, :, 0] = 2.0 ** np.floor(np.log2(5.0 / unit * dim ** 0.5))  # scores of up to 5
    s = Sequence(kind, dtype, 2, 2, dim, keys, values, k_exp, v_exp, q)
    other = s.pool.scales[:, 1 - plane].clone()
    s.pool.scales[s.pool.scales == (1 if byte == 0 else 254)] = byte
    assert (s.pool.scales[:, plane] == byte).sum() >= 2 * tiles and torch.equal(s.pool.scales[:, 1 - plane], other)
    got = s.pool.dequantize(0, torch.from_numpy(s.table[0]).long().to(DEV))[plane][:n].double().cpu().numpy()
    np.testing.assert_array_equal(got, s.cache.values(0, plane, s.at))
    s.check(rng)


@pytest.mark.parametrize("byte", [0, 255])
def test_write_joins_a_tile_whose_scale_byte_is_outside_its_range(byte) -> None:
    rng = np.random.default_rng(75)
    n, new = 5, 6
    codes = np.zeros((1, 2, 1, 2, 16, 64))
    codes[:, :, :, :, :n] = oracle.round_e4m3(np.clip(rng.standard_normal((n, 64)) * 90, -448, 448))
    cache = oracle.Cache(codes, np.full((1, 2, 1, 2), -126 if byte == 0 else 127))
    pool = kv8.Kv8Pool(helpers.pack(codes, 16).to(DEV), torch.full((1, 2, 1, 2, 1), byte, dtype=torch.uint8, device=DEV))
    k, v = (helpers.values(rng, "f32", new, 2, 64) for _ in range(2))
    if byte == 0:  # far below the range of normal tiles: what was there still counts
        k, v = k * 2.0 ** -120, v * 2.0 ** -120
    at = torch.arange(n, n + new)
    kv8.write_raw(None, k.to(DEV), v.to(DEV), None, pool, 0, at.to(DEV), at.int().to(DEV), None, None, 0, None, None)
    cache.write(0, at.numpy(), k.numpy(), v.numpy())
    helpers.same_cache(pool, cache)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("f32", 128), ("bf16", 96)])
@pytest.mark.parametrize("size", [21.7, 22.3, 23.4, 24.6, 25.5, 26.2, 27.8, 28.5, 31.1, 60.0, 110.0])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_of_any_size_pick_the_largest(kind, dtype, dim, size, sign) -> None:
    """Scores of up to +-2^size, whose gaps are far past what any computation is off by: the result is the value of the
    largest, and the mean of both where two are the same."""
    rng = np.random.default_rng(76)
    n, tiles = 600, 38
    first = np.where(sign > 0, rng.uniform(0.0, 200.0, n), rng.uniform(-448.0, -300.0, n))
    best, last = (448.0, 0.0) if sign > 0 else (-200.0, -440.0)
    first[37] = first[520] = best
    first[-40:] = np.minimum(first[-40:], last if sign < 0 else 200.0)
    keys, values = line(rng, n, 2, dim, first)
    q = np.zeros((1 if kind == "decode" else 40, 2, dim))
    q[:, :, 0] = 2.0 ** (size - 8.8) * dim ** 0.5 * 16 * np.log(2.0)  # a key's code is 2^8.8 at most, over 16
    s = Sequence(kind, dtype, 2, 2, dim, keys, values, np.full(tiles, -4), np.full(tiles, -6), q)
    got = (s.run(*s.new_token(rng, key=-28.0 if sign < 0 else 0.0)) if kind == "decode" else s.run()).double().cpu()
    v = s.cache.values(0, 1, s.at)
    want, size = (v[37] + v[520]) / 2, (np.abs(v[37]) + np.abs(v[520])) / 2
    # Probabilities leave 2^-11 (fp32 models 2^-23) of each term, which may cancel; products, sum, division and result
    # round once each.
    bound = (2.0 ** -8 * np.abs(want) + 2.0 ** -11 * size if dtype == "bf16" else (2.0 ** -23 + 4 * TINY) * size)
    helpers.close(got, np.broadcast_to(want, got.shape), np.broadcast_to(bound, got.shape) + 2.0 ** -100)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("f32", 128)])
def test_scores_of_minus_infinity_count_for_nothing(kind, dtype, dim) -> None:
    """Keys whose scores overflow to minus infinity before others that do not.

    They are some -2^128.4 (decode takes a query in parts, the second up to 2^-4 of the first and of either sign: from
    2^132 on both overflow, and minus and plus infinity make NaN; no score exists in fp32 there)."""
    rng = np.random.default_rng(77)
    n, tiles = 600, 38
    first = np.full(n, -448.0)
    first[300:] = 0.0
    keys, values = line(rng, n, 1, dim, first)
    k_exp = np.where(np.arange(tiles) < 18, 60, -4)
    q = np.zeros((1 if kind == "decode" else 40, 1, dim))
    q[:, :, 0] = 2.0 ** 128.4 / (2.0 ** 68.8 * np.log2(np.e) * dim ** -0.5)
    s = Sequence(kind, dtype, 1, 1, dim, keys, values, k_exp, np.full(tiles, -6), q)
    got = (s.run(*s.new_token(rng)) if kind == "decode" else s.run()).double().cpu()
    v = s.cache.values(0, 1, s.at)
    end = np.arange(n - s.new, n)
    want = np.stack([v[300:e + 1].mean(0) for e in end])
    np.testing.assert_allclose(got.numpy(), want, rtol=0, atol=2.0 ** -8 * np.abs(want).max() + 2.0 ** -11 * np.abs(v).mean())


@pytest.mark.parametrize("kind", ["decode", "prefill"])
@pytest.mark.parametrize("dim", [64, 128])
def test_fp32_probabilities_are_as_exact_as_their_scores(kind, dim) -> None:
    """Few keys whose scores are exact: what is left is the exponential and a few roundings.

    Scores below the largest lie within 2 of it (in log2), so the exponential's argument rounds by 2^-24 at most (2^-21
    and more if something were added to it first), which moves a probability by ln 2 of that; the scale's own
    rounding and the product by it move the argument by 2^-23 of 4, all the same way; the exponential is within an
    ulp, 2^-23. Parts leave 2^-23; six more roundings of sums, products and the division. Of |v|, weighed.
    """
    rng = np.random.default_rng(78)
    n = 16
    keys, values = line(rng, n, 2, dim, rng.integers(0, 9, n) * 8.0)  # 0..64 over 16
    q = np.zeros((1 if kind == "decode" else 12, 2, dim))
    q[:, :, 0] = 0.5 * dim ** 0.5 if dim == 64 else 4.0
    got, want, mass = [], [], []
    for seed in range(40):
        values = oracle.round_e4m3(np.clip(rng.standard_normal((n, 2, dim)) * 90, -448, 448))
        s = Sequence(kind, "f32", 2, 2, dim, keys, values, np.full(1, -4), np.full(1, -6), q, new=12)
        got.append((s.run(*s.new_token(rng)) if kind == "decode" else s.run()).double().cpu().numpy())
        k, v = (s.cache.values(0, plane, s.at) for plane in (0, 1))
        end = np.arange(n - s.new, n)
        w, _ = expect(s.q.double().cpu().numpy(), k, v, end, s.scale, **numerics(kind, "f32", dim, n))
        m, _ = expect(s.q.double().cpu().numpy(), k, np.abs(v), end, s.scale, **numerics(kind, "f32", dim, n))
        want.append(w), mass.append(m)
    off = np.abs(np.array(got) - want) / np.array(mass)
    assert off.max() <= (0.7 * 2.0 ** -24 + 4 * 2.0 ** -23 * 0.7 + 2.0 ** -23 + 2.0 ** -23 + 6 * TINY) * 2
    # A rounding is some 0.4 * 2^-24 in the mean square. Those of single keys average out; three do not: the sum's, the
    # division's and the result's.
    assert np.sqrt((off ** 2).mean()) <= 0.75 * 2.0 ** -24
