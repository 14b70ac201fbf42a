"""The packed and int8-cache ops at the edges of what their documentation allows: starts in no order, long sequences,
strides, values of very different sizes."""
from __future__ import annotations

import numpy as np
import pytest
import seq_oracle as so
from test_gpu_kv_q8 import UNIT_P as Q8_UNIT_P
from test_gpu_kv_q8 import Cache, assert_within, attend
from test_gpu_packed import TYPES, UNIT, UNIT_P, Packed, as_type, code, from_type, status

pytestmark = pytest.mark.gpu

# Descending somewhere, though all sequences together have no more rows than the buffer's 100.
DESCENDING = [[0, 40, 10, 60], [0, 60, 59, 60], [5, 0, 50, 60], [0, 30, 60, 20]]


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("starts", DESCENDING)
def test_packed_descending_starts_with_rows_to_spare_run_nothing(lz, device, suite, starts, qt, kt):
    c = Packed(lz, device, suite, 64, 4, 2, [40, 20, 20], [40, 20, 20], qt, kt, tail=20)
    b = c.buffers()
    status(lz, device)
    b[4].Write(np.array(starts, np.int32))
    c.call(b)
    assert status(lz, device) == 2
    assert np.all(c.read(b) == 7.0)
    b[4].Write(c.q_starts)  # and the next call is right
    c.call(b)
    c.check(c.read(b))
    assert status(lz, device) == 0
    for x in b:
        x.Dispose()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("starts", DESCENDING)
def test_q8_descending_starts_with_rows_to_spare_run_nothing(lz, device, suite, starts, dt):
    rng = np.random.default_rng(30)
    c = Cache(lz, device, suite, 3, 128, 2, 64, 32, rng, scale=0.01)
    st, le = c.int_buffer(starts), c.int_buffer([128, 100, 60])
    x = as_type(np.full(100 * 256, 3.0), dt)[0]
    status(lz, device)
    with lz.SharedBuffer.from_array(device, x, code(lz, dt)) as qb, lz.SharedBuffer.from_array(device, x, code(lz, dt)) as ob:
        suite.Attention.ExecuteQ8(device, qb, *c.buffers, ob, st, le, 64, 4, 2, 32, 128, 3, 100)
        assert status(lz, device) == 2
        assert np.all(from_type(ob.ToArray(), dt) == 3.0)
    assert_within(*attend(lz, device, suite, c, 4, [40, 20, 30], [128, 100, 60], dt))
    assert status(lz, device) == 0
    for b in (st, le):
        b.Dispose()
    c.dispose()


@pytest.mark.parametrize("starts", [[50, 60, 10, 20], [64, 70, 3, 3]])
def test_load_touches_nothing_in_front_of_a_sequence(lz, device, suite, starts):
    # The search for a row's sequence counts the starts up to it: of starts that descend it may name one that begins
    # behind the row, whose slots in front of its position lie outside the cache.
    rng = np.random.default_rng(31)
    c = Cache(lz, device, suite, 3, 64, 1, 64, 32, rng)
    st, po = c.int_buffer(starts), c.int_buffer([1, 0, 2])
    out = [lz.SharedBuffer.from_array(device, np.full(100 * 64, 9, np.float32)) for _ in range(2)]
    status(lz, device)
    suite.KvCacheQ8.Load(device, *c.buffers, *out, st, po, 1, 64, 32, 64, 3, 100)
    assert status(lz, device) == 2
    for w in range(2):
        got = out[w].ToArray().reshape(100, 64)
        want = np.full((100, 64), 9, np.float32)
        for i in range(3):  # rows of a sequence as its own starts have them, or left as they were
            for t in range(starts[i], max(starts[i], min(starts[i + 1], 100))):
                if np.any(got[t] != 9):
                    want[t] = so.values(c.codes[w][i], c.scales[w][i], 32)[po.ToArray()[i] + t - starts[i], 0].astype(np.float32)
        np.testing.assert_array_equal(got, want)
    for x in (st, po, *out):
        x.Dispose()
    c.dispose()


@pytest.mark.parametrize("starts", [*DESCENDING, [0, 50, 10, 60], [90, 95, 99, 0]])
def test_store_and_load_report_descending_starts(lz, device, suite, starts):
    rng = np.random.default_rng(32)
    c = Cache(lz, device, suite, 3, 128, 1, 64, 32, rng)
    st, po = c.int_buffer(starts), c.int_buffer([0, 0, 0])
    x = [lz.SharedBuffer.from_array(device, rng.standard_normal(100 * 64).astype(np.float32)) for _ in range(2)]
    status(lz, device)
    suite.KvCacheQ8.Load(device, *c.buffers, *x, st, po, 1, 64, 32, 128, 3, 100)
    assert status(lz, device) == 2
    suite.KvCacheQ8.Store(device, *x, *c.buffers, st, po, 1, 64, 32, 128, 3, 100)
    assert status(lz, device) == 2
    for b in (st, po, *x):
        b.Dispose()
    c.dispose()


def test_store_and_load_look_at_every_start(lz, device, suite):
    # one descending pair among more starts than a CTA has threads
    count = 1500
    c = Cache(lz, device, suite, count, 8, 1, 64, 32)
    x = [lz.SharedBuffer(device, lz.F32, 2 * count * 64) for _ in range(2)]
    po = c.int_buffer(np.zeros(count))
    for at in (None, 1, 700, count - 1):
        starts = np.arange(count + 1)
        if at is not None:
            starts[at] += 2
        st = c.int_buffer(starts)
        status(lz, device)
        for op, args in (("Store", (*x, *c.buffers)), ("Load", (*c.buffers, *x))):
            getattr(suite.KvCacheQ8, op)(device, *args, st, po, 1, 64, 32, 8, count, 2 * count)
            assert status(lz, device) == (0 if at is None else 2)
        st.Dispose()
    for b in (po, *x):
        b.Dispose()
    c.dispose()


# ----------------------------------------------------------------------------------------------
# Long sequences
# ----------------------------------------------------------------------------------------------

def check_long(c, got, floor_p=2.0 ** -38):
    """Packed.check, with what the MMA cuts off O for 16-bit queries: 5 * 2^-23 of the sum at most for each of the 512
    steps that it is summed over, and no more than 2 * 2^-23 of them on average for keys alike."""
    out, spread, dot, mass = c.want()
    bound = so.attention_bound(out, spread, dot, mass, c.hd, UNIT_P[c.qt], UNIT[c.qt], floor_p)
    if c.qt != "f32":
        bound += 1024 * 2.0 ** -23 * (np.abs(out) + spread)
    err = np.abs(got - out)
    assert np.all(err <= bound), f"{(err / bound).max():.3g} of the bound, max err {err.max():.3g}"
    return out


# Values of one sign, so that truncated sums add up; keys enough for them to pass half a step of the result's type.
@pytest.mark.parametrize("qt,kt,m,hd,nh", [("f16", "f16", 300000, 64, 2), ("f16", "f16", 300000, 128, 1),
                                           ("bf16", "bf16", 1200000, 64, 1), ("f32", "f16", 300000, 128, 1),
                                           ("f32", "bf16", 300000, 64, 2)])
def test_sums_over_many_keys_do_not_drift(lz, device, suite, qt, kt, m, hd, nh):
    def edit(q, k, v):
        q *= 0.1
        v[:] = np.abs(v) + 0.5

    c = Packed(lz, device, suite, hd, nh, 1, [2], [m], qt, kt, edit=edit)
    check_long(c, c.run())


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("hd,nh", [(64, 2), (128, 1)])
def test_many_small_weights_beside_a_large_one(lz, device, suite, hd, nh, qt, kt):
    # One key at about 2^26 times the weight of 131,071 others, its value 0: what is left is the sum of the small ones.
    # f16 weights keep steps of 2^-24 under a factor of 2^7 at least: half a step is 2^-32 of the largest weight.
    def edit(q, k, v):
        q[:, 0::hd] = 16.0
        q[:, 1:hd] *= 0.5
        k[:, 0] = 0
        k[0] = 0
        k[0, 0] = 26 * np.log(2) * np.sqrt(hd) / 16
        v[:] = np.abs(v) + 0.5
        v[0] = 0

    c = Packed(lz, device, suite, hd, nh, 1, [2], [131072], qt, kt, edit=edit)
    out = check_long(c, c.run(), floor_p=2.0 ** -32 if qt == "f16" else 2.0 ** -38)
    assert np.all(out > 2.0 ** -11)


@pytest.mark.parametrize("qt,kt,m", [("f16", "f16", 262144), ("bf16", "bf16", 1048576), ("f32", "f16", 262144)])
def test_many_small_keys_behind_a_large_one_in_the_sum(lz, device, suite, qt, kt, m):
    # The first key's share of O is about 1, each other's below what a truncated sum next to it holds: lost in the first
    # 512 steps alone (5 * 2^-23 of the sum for each of them at most), not in all.
    def edit(q, k, v):
        q[:, 0] = 16.0
        q[:, 1:] *= 0.5
        k[:, 0] = 0
        k[0] = 0
        k[0, 0] = 25.5 * np.log(2) * 8 / 16
        v[:] = np.abs(v) + 0.5
        v[0] = 1

    c = Packed(lz, device, suite, 64, 1, 1, [1], [m], qt, kt, edit=edit)
    out, spread, dot, mass = c.want()
    bound = so.attention_bound(out, spread, dot, mass, 64, UNIT_P[qt], UNIT[qt], 2.0 ** -32 if qt == "f16" else 2.0 ** -38)
    if qt != "f32":
        bound += 512 * 5 * 2.0 ** -23 * out
    err = np.abs(c.run() - out)
    assert np.all(err <= bound), f"{(err / bound).max():.3g} of the bound, max err {err.max():.3g}"


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("hd,nh,nkv,m", [(64, 4, 2, 16384), (128, 3, 3, 16385), (128, 2, 1, 16512), (64, 3, 1, 40000)])
def test_few_rows_behind_a_long_prefix(lz, device, suite, hd, nh, nkv, m, qt, kt):
    # on both sides of the 128 tiles of one sum, with a reference that moves late: the last keys are the largest
    def edit(q, k, v):
        k *= np.linspace(0.2, 3.0, k.shape[0])[:, None]

    c = Packed(lz, device, suite, hd, nh, nkv, [3, 1], [m, 130], qt, kt, edit=edit)
    check_long(c, c.run())


@pytest.mark.parametrize("qt,kt", [("f16", "f16"), ("bf16", "bf16")])
def test_a_carry_of_rows_that_saw_nothing_or_no_number(lz, device, suite, qt, kt):
    # a key that is no number in the first sum shows in every row; scores of minus infinity alone there weigh nothing
    m, hd = 20000, 64
    for bad in (np.nan, -np.inf):
        def edit(q, k, v):
            q[:, 0] = 1.0
            k[:16384, 0] = bad

        c = Packed(lz, device, suite, hd, 1, 1, [5], [m], qt, kt, edit=edit)
        with np.errstate(all="ignore"):
            got = c.run()
        if np.isnan(bad):
            assert not np.isfinite(got).any()
            continue
        o, *errs = so.attention(c.qv, c.kv[16384:], c.vv[16384:], np.arange(m - 16384 - 5, m - 16384), 1, 1)
        assert np.all(np.abs(got - o) <= so.attention_bound(o, *errs, hd, UNIT_P[qt], UNIT[qt], 2.0 ** -32))


def test_same_bits_of_a_long_sequence_replayed(lz, device, suite):
    c = Packed(lz, device, suite, 128, 4, 2, [200, 300], [20000, 33000], "bf16", "bf16")
    b = c.buffers()
    c.call(b)
    first = b[3].ToArray()
    for _ in range(2):
        device.BeginRecording()
        c.call(b)
        device.EndRecording()
        np.testing.assert_array_equal(b[3].ToArray(), first)
    for x in b:
        x.Dispose()


# ----------------------------------------------------------------------------------------------
# Attention over the int8 cache
# ----------------------------------------------------------------------------------------------

def attend_rows(lz, device, suite, c, nh, q, n, lengths, dt, stride=0):
    """ExecuteQ8 of the rows q [sum(n), nh * hd] (strided by `stride` elements where given); (got, want, bound)."""
    rows, width = q.shape
    qs, qv = as_type(q, dt)
    held = qs if not stride else np.pad(qs, ((0, 0), (0, stride - width)))
    st, le = c.int_buffer(np.concatenate([[0], np.cumsum(n)])), c.int_buffer(lengths)
    with lz.SharedBuffer.from_array(device, held, code(lz, dt)) as qb, lz.SharedBuffer(device, code(lz, dt), rows * width) as ob:
        suite.Attention.ExecuteQ8(device, qb, *c.buffers, ob, st, le, c.hd, nh, c.nkv, c.block, c.max_seq, c.count, rows, stride)
        got = from_type(ob.ToArray(), dt).reshape(rows, nh, c.hd)
    for x in (st, le):
        x.Dispose()
    want, bound, a = np.zeros(got.shape), np.zeros(got.shape), 0
    for i, (m, length) in enumerate(zip(n, lengths)):
        k, v = (so.values(c.codes[w][i][:length], c.scales[w][i], c.block).reshape(length, -1) for w in range(2))
        o, *errs = so.attention(qv[a:a + m], k, v, np.arange(length - m, length), nh, c.nkv)
        want[a:a + m], bound[a:a + m] = o, so.attention_bound(o, *errs, c.hd, Q8_UNIT_P[dt], UNIT[dt])
        a += m
    return got, want, bound


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,nh,n", [(128, 4, [1, 1]), (64, 14, [1, 3])])
@pytest.mark.parametrize("loud,key", [(1e2, 0), (1e3, 0), (1e4, 0), (1e3, 1)])
def test_q8_queries_with_a_loud_channel(lz, device, suite, loud, key, hd, nh, n, dt):
    # A query channel far above the others where the keys' codes are 0 or tiny: the others make the score, and keep
    # the accuracy of a sum in f32 that never met the loud one. Queries enter as integers of 31 bits of the largest (bf16:
    # 23): at 1e4 the others of size 1 are off by 2^-17 each at most, on terms of random sign; the bound has (hd / 8 + 4)
    # 2^-23 of the sum of all magnitudes (bf16: 2^-9, less than half a step of its values, and its weights' 2^-11).
    rng = np.random.default_rng(40)
    c = Cache(lz, device, suite, 2, 300, 2, hd, 64, rng, scale=0.01)
    c.codes[0][..., 5] = key * rng.integers(-1, 2, c.codes[0][..., 5].shape)
    c.buffers[0].Write(c.codes[0])
    q = rng.standard_normal((sum(n), nh * hd))
    q[:, 5::hd] = loud
    assert_within(*attend_rows(lz, device, suite, c, nh, q, n, [300, 170], dt))
    c.dispose()


@pytest.mark.parametrize("length", [20, 3000])  # one part, and parts that are joined
def test_q8_a_row_whose_scores_are_all_minus_infinity(lz, device, suite, length):
    # it sees slots, so it is not a row of zeros: its scores pass the range of f32
    rng = np.random.default_rng(41)
    c = Cache(lz, device, suite, 2, 3000, 2, 64, 32, rng, scale=0.01)
    c.codes[0][:] = 100
    c.buffers[0].Write(c.codes[0])
    st, le = c.int_buffer([0, 2, 3]), c.int_buffer([length, 0])
    q = rng.standard_normal((3, 4, 64)).astype(np.float32)
    q[0, 1] = -3e38
    with lz.SharedBuffer.from_array(device, q) as qb, lz.SharedBuffer(device, lz.F32, q.size) as ob:
        suite.Attention.ExecuteQ8(device, qb, *c.buffers, ob, st, le, 64, 4, 2, 32, 3000, 2, 3)
        got = ob.ToArray().reshape(q.shape)
    assert np.all(np.isnan(got[0, 1]))
    got[0, 1] = 1
    assert np.all(np.isfinite(got)) and not got[2].any()
    for x in (st, le):
        x.Dispose()
    c.dispose()


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("count,length,nh,nkv,hd", [(1, 20000, 8, 1, 128), (3, 6000, 14, 2, 64), (40, 700, 8, 8, 128)])
def test_q8_long_contexts_of_16_bit_queries(lz, device, suite, count, length, nh, nkv, hd, dt):
    rng = np.random.default_rng(length)
    c = Cache(lz, device, suite, count, length, nkv, hd, 64, rng, scale=0.01)
    lengths = [max(1, length - 997 * i % length) for i in range(count)]
    assert_within(*attend(lz, device, suite, c, nh, [1] * count, lengths, dt))
    c.dispose()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,nh,nkv,block", [(128, 28, 4, 64), (64, 9, 3, 128)])
def test_q8_several_strided_rows_a_sequence(lz, device, suite, hd, nh, nkv, block, dt):
    rng = np.random.default_rng(42)
    c = Cache(lz, device, suite, 4, 260, nkv, hd, block, rng, scale=0.01)
    n, lengths = [5, 0, 17, 9], [5, 77, 260, 3]  # the last has rows that see nothing
    q = rng.standard_normal((sum(n), nh * hd))
    got, want, bound = attend_rows(lz, device, suite, c, nh, q, n, lengths, dt, stride=nh * hd + 24)
    assert_within(got, want, bound)
    assert not got[-9:-3].any()
    c.dispose()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("which", [0, 1])  # scales of keys, of values
def test_q8_a_scale_that_is_not_finite_shows_in_its_heads_alone(lz, device, suite, which, bad):
    rng = np.random.default_rng(43)
    c = Cache(lz, device, suite, 2, 300, 2, 64, 32, rng, scale=0.01)
    before, *_ = attend(lz, device, suite, c, 6, [1, 2], [300, 200], "f32")
    c.scales[which][1, 3, 1] = bad  # a block that both rows of the second sequence see, of the second KV head
    c.buffers[2 + which].Write(c.scales[which])
    with np.errstate(all="ignore"):
        after, *_ = attend(lz, device, suite, c, 6, [1, 2], [300, 200], "f32")
    assert not np.isfinite(after[1:, 3:]).any()
    after[1:, 3:] = before[1:, 3:]
    np.testing.assert_array_equal(after, before)
    c.dispose()


def test_q8_accuracy_behind_offsets_past_32_bits(lz, device, suite):
    # The second sequence's codes start behind 2^31 bytes; 2.2 million slots score 0 with a value of 0, 150 are stored.
    max_seq, nkv, hd, block, n = 2_200_000, 8, 128, 128, 150
    assert max_seq * nkv * hd > 2 ** 31
    blocks, pos = -(-max_seq // block), max_seq - n
    rng = np.random.default_rng(44)
    bufs = [lz.SharedBuffer(device, lz.I8, 2 * max_seq * nkv * hd) for _ in range(2)]
    bufs += [lz.SharedBuffer(device, lz.F32, 2 * blocks * nkv) for _ in range(2)]
    k, v = (rng.standard_normal((n, nkv * hd)).astype(np.float32) for _ in range(2))
    ints = [lz.SharedBuffer.from_array(device, np.array(x, np.int32)) for x in ([0, 0, n], [0, pos], [0, max_seq], [0, 0, 1])]
    kb, vb, ko, vo = (lz.SharedBuffer.from_array(device, x) for x in (k, v, k * 0, v * 0))
    suite.KvCacheQ8.Store(device, kb, vb, *bufs, *ints[:2], nkv, hd, block, max_seq, 2, n)
    suite.KvCacheQ8.Load(device, *bufs, ko, vo, *ints[:2], nkv, hd, block, max_seq, 2, n)
    q = (rng.standard_normal((1, nkv * hd)) * 8).astype(np.float32)
    with lz.SharedBuffer.from_array(device, q) as qb, lz.SharedBuffer(device, lz.F32, nkv * hd) as ob:
        suite.Attention.ExecuteQ8(device, qb, *bufs, ob, ints[3], ints[2], hd, nkv, nkv, block, max_seq, 2, 1)
        got = ob.ToArray().reshape(nkv, hd)
    kk, vv = (b.ToArray().reshape(n, nkv, hd).astype(np.float64) for b in (ko, vo))
    s = np.einsum("jhd,hd->hj", kk, q.reshape(nkv, hd).astype(np.float64)) / np.sqrt(hd)
    w = np.exp(s)
    p = w / (w.sum(1, keepdims=True) + (max_seq - n))
    out, spread = np.einsum("hj,jhd->hd", p, vv), np.sqrt(np.einsum("hj,jhd->hd", p * p, vv * vv))
    dot = np.abs(kk * q.reshape(nkv, hd)).sum(2).max(0) / np.sqrt(hd)
    bound = so.attention_bound(out, spread, dot, np.abs(vv).sum(0), hd, Q8_UNIT_P["f32"], UNIT["f32"])
    # and the result is one of weights that were summed in f32 over a run: 2.2 million / (148 SMs x 12 warps / 8 heads)
    # slots a warp are 310 tiles, of which a rounding of 2^-24 each can only shrink or grow all outputs alike
    assert_within(got, out, bound + 310 * 2.0 ** -24 * np.abs(out))
    for x in (*ints, kb, vb, ko, vo, *bufs):
        x.Dispose()


# ----------------------------------------------------------------------------------------------
# Strides, and rows past 2^31 elements
# ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,nkv,block", [(64, 2, 32), (128, 3, 128)])
def test_store_and_load_of_strided_rows(lz, device, suite, hd, nkv, block, dt):
    rng = np.random.default_rng(45)
    c = Cache(lz, device, suite, 3, 200, nkv, hd, block)
    width, strides = nkv * hd, (nkv * hd + 8, nkv * hd + 40)
    n, pos = [130, 0, 37], [3, 0, 100]
    rows = sum(n)
    stored, values = zip(*(as_type(rng.standard_normal((rows, width)), dt) for _ in range(2)))
    st, po = c.int_buffer(np.concatenate([[0], np.cumsum(n)])), c.int_buffer(pos)
    x = [lz.SharedBuffer.from_array(device, np.pad(y, ((0, 0), (0, s - width)), constant_values=7), code(lz, dt))
         for y, s in zip(stored, strides)]
    out = [lz.SharedBuffer(device, code(lz, dt), rows * s) for s in strides]
    suite.KvCacheQ8.Store(device, *x, *c.buffers, st, po, nkv, hd, block, 200, 3, rows, *strides)
    c.store_model(*values, n, pos)
    c.check()
    suite.KvCacheQ8.Load(device, *c.buffers, *out, st, po, nkv, hd, block, 200, 3, rows, *strides)
    for w in range(2):
        got = from_type(out[w].ToArray(), dt).reshape(rows, strides[w])
        want = np.concatenate([so.values(c.codes[w][i], c.scales[w][i], block)[p:p + m] for i, (m, p) in enumerate(zip(n, pos))])
        want = from_type(as_type(want.reshape(rows, width).astype(np.float32), dt)[0], dt)
        np.testing.assert_array_equal(got[:, :width], want)
        assert not got[:, width:].any()
    assert status(lz, device) == 0
    for b in (st, po, *x, *out):
        b.Dispose()
    c.dispose()


@pytest.mark.parametrize("qt,kt", TYPES)
def test_packed_strides_of_their_own(lz, device, suite, qt, kt):
    hd, nh, nkv, n, m = 64, 6, 2, [90, 41, 3], [90, 141, 700]
    c = Packed(lz, device, suite, hd, nh, nkv, n, m, qt, kt)
    strides = [nh * hd + 8, nkv * hd + 16, nkv * hd + 40, nh * hd + 24]
    wide = [np.pad(x, ((0, 0), (0, s - x.shape[1]))) for x, s in zip((c.q, c.k, c.v), strides)]
    b = [lz.SharedBuffer.from_array(device, x, code(lz, t)) for x, t in zip(wide, (qt, kt, kt))]
    b += [lz.SharedBuffer(device, code(lz, qt), c.tokens * strides[3])]
    b += [lz.SharedBuffer.from_array(device, x) for x in (c.q_starts, c.kv_starts)]
    suite.Attention.ExecutePacked(device, *b, hd, nh, nkv, 3, c.tokens, c.kv_tokens, *strides)
    got = from_type(b[3].ToArray(), qt).reshape(c.tokens, strides[3])
    assert not got[:, nh * hd:].any()
    np.testing.assert_array_equal(got[:, :nh * hd].reshape(c.tokens, nh, hd), c.run())
    for x in b:
        x.Dispose()


@pytest.mark.parametrize("qt,kt", [("f16", "f16"), ("f32", "bf16")])
def test_packed_rows_past_2_to_the_31_elements(lz, device, suite, qt, kt):
    c = Packed(lz, device, suite, 64, 2, 1, [100, 40], [100, 40], qt, kt)
    stride, rows = 1 << 24, 140
    assert (rows - 1) * stride > 2 ** 31
    b = []
    for x, t in ((c.q, qt), (c.k, kt), (c.v, kt), (None, qt)):
        b.append(lz.SharedBuffer(device, code(lz, t), (rows - 1) * stride + 128))
        for r in range(rows if x is not None else 0):
            with b[-1].View(r * stride, x.shape[1]) as row:
                row.Write(x[r])
    b += [lz.SharedBuffer.from_array(device, x) for x in (c.q_starts, c.kv_starts)]
    suite.Attention.ExecutePacked(device, *b, 64, 2, 1, 2, rows, rows, *[stride] * 4)
    got = []
    for r in range(rows):
        with b[3].View(r * stride, 128) as row:
            got.append(from_type(row.ToArray(), qt))
    np.testing.assert_array_equal(np.stack(got).reshape(rows, 2, 64), c.run())
    for x in b:
        x.Dispose()
