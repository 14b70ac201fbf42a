"""The int8 KV cache: store and load bit for bit against their definition, attention over it against a plain 64-bit
form, and the ops together as a server uses them."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import seq_oracle as so
from test_gpu_packed import I32_MAX, I32_MIN, UNIT, as_type, code, from_type, status

pytestmark = pytest.mark.gpu


class Cache:
    def __init__(self, lz, device, suite, count, max_seq, nkv, hd, block, rng=None, scale=0.02):
        self.lz, self.device, self.suite = lz, device, suite
        self.count, self.max_seq, self.nkv, self.hd, self.block = count, max_seq, nkv, hd, block
        self.blocks = -(-max_seq // block)
        shape, sshape = (count, max_seq, nkv, hd), (count, self.blocks, nkv)
        self.codes = [np.zeros(shape, np.int8) for _ in range(2)]
        self.scales = [np.zeros(sshape, np.float32) for _ in range(2)]
        if rng is not None:
            self.codes = [rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2)]
            self.scales = [(rng.random(sshape) * scale + scale / 2).astype(np.float32) for _ in range(2)]
        self.buffers = [lz.SharedBuffer.from_array(device, x) for x in (*self.codes, *self.scales)]

    def read(self):
        got = [b.ToArray() for b in self.buffers]
        return [g.reshape(w.shape) for g, w in zip(got, (*self.codes, *self.scales))]

    def dispose(self):
        for b in self.buffers:
            b.Dispose()

    def int_buffer(self, x):
        return None if x is None else self.lz.SharedBuffer.from_array(self.device, np.asarray(x, np.int32))

    def store(self, k, v, dt, n, positions, starts="sum"):
        """k, v: [rows, nkv * hd] storage arrays."""
        st = self.int_buffer(np.concatenate([[0], np.cumsum(n)]) if isinstance(starts, str) else starts)
        po = self.int_buffer(positions)
        kb, vb = (self.lz.SharedBuffer.from_array(self.device, x, code(self.lz, dt)) for x in (k, v))
        self.suite.KvCacheQ8.Store(self.device, kb, vb, *self.buffers, st, po, self.nkv, self.hd, self.block,
                                   self.max_seq, self.count, k.shape[0])
        self.device.Synchronize()
        for x in (st, po, kb, vb):
            if x is not None:
                x.Dispose()

    def store_model(self, k, v, n, positions):
        a = 0
        for i, (rows, pos) in enumerate(zip(n, positions)):
            for w, x in enumerate((k, v)):
                so.store(x[a:a + rows].reshape(rows, self.nkv, self.hd).astype(np.float64), self.codes[w][i],
                         self.scales[w][i], pos, self.block)
            a += rows

    def check(self):
        got = self.read()
        for g, w in zip(got, (*self.codes, *self.scales)):
            np.testing.assert_array_equal(g, w)


def rows_of(rng, n, width, dt, gain=1.0):
    pairs = [as_type(rng.standard_normal((n, width)) * gain * np.exp(0.5 * rng.standard_normal(width)), dt)
             for _ in range(2)]
    return [p[0] for p in pairs], [p[1] for p in pairs]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("hd,nkv", [(64, 2), (128, 3)])
def test_store_matches_the_definition(lz, device, suite, hd, nkv, block, dt):
    rng = np.random.default_rng(hd + block)
    c = Cache(lz, device, suite, 6, 300, nkv, hd, block)
    # prompts (one empty), then single tokens, then runs that start inside a block, with growing and shrinking rows
    plans = [([300, 1, 0, 129, 64, 31], [0, 0, 0, 0, 0, 0], 1.0), ([0, 1, 1, 1, 1, 1], [0, 1, 0, 129, 64, 31], 3.0),
             ([0, 5, 40, 7, 100, 1], [0, 2, 1, 130, 65, 32], 0.3), ([7, 9, 3, 7, 1, 9], [290, 5, 40, 100, 0, 20], 2.0),
             ([1, 1, 1, 1, 1, 1], [299, 14, 43, 107, 1, 29], 1.5)]
    for step, (n, pos, gain) in enumerate(plans):
        (k, v), (kv, vv) = rows_of(rng, sum(n), nkv * hd, dt, gain)
        single = all(x == 1 for x in n)
        c.store(k, v, dt, n, pos, starts=None if single else "sum")
        c.store_model(kv, vv, n, pos)
        c.check()
        c.store(k, v, dt, n, pos)  # the same rows again change nothing
        c.check()
    assert status(lz, device) == 0
    c.dispose()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_store_next_to_halves(lz, device, suite, dt):
    # x = (j + 1/2) * scale lands on ties; neighbours one ulp off do not
    hd, block = 64, 32
    c = Cache(lz, device, suite, 1, 64, 1, hd, block)
    rng = np.random.default_rng(0)
    k = np.zeros((64, hd), np.float32)
    for r in range(64):
        top = np.float32(2.0 ** rng.integers(-60, 60)) * np.float32(127 if r < 32 else rng.integers(1, 127))
        k[r] = (rng.integers(-127, 127, hd) + 0.5).astype(np.float32) * np.float32(top / 127)
    k[:32] = (rng.integers(-126, 126, (32, hd)) + 0.5).astype(np.float32) * np.float32(0.25)
    k[0, 0] = 127 * 0.25
    k[1::3] = np.nextafter(k[1::3], np.float32(np.inf))
    ks, kv = as_type(k, dt)
    c.store(ks, ks, dt, [64], [0])
    c.store_model(kv, kv, [64], [0])
    c.check()
    c.dispose()


def test_store_extremes(lz, device, suite):
    # zeros, denormals, the largest numbers, infinities and NaN, each in a block of its own
    hd, block = 64, 32
    c = Cache(lz, device, suite, 1, 8 * block, 2, hd, block)
    rng = np.random.default_rng(1)
    x = rng.standard_normal((8 * block, 2 * hd)).astype(np.float32)
    x[0:32] = 0
    x[32:64] *= np.float32(1e-44)
    x[64:96] *= np.float32(1e-38)
    x[96:128] *= np.float32(3e37)
    x[130, 5] = np.inf
    x[163, 70] = np.nan
    x[192:224] *= np.float32(1e-42)
    with np.errstate(all="ignore"):
        c.store(x, x, "f32", [256], [0])
        c.store_model(x, x, [256], [0])
        c.check()
        one = np.full((1, 2 * hd), 1e30, np.float32)
        for pos in (20, 50, 150, 180, 200):  # into the kept part of each kind of block
            c.store(one, one, "f32", [1], [pos])
            c.store_model(one, one, [1], [pos])
            c.check()
    c.dispose()


def test_store_outside_the_cache(lz, device, suite):
    c = Cache(lz, device, suite, 3, 70, 1, 64, 32)
    rng = np.random.default_rng(2)
    (k, v), (kv, vv) = rows_of(rng, 30, 64, "f32")
    status(lz, device)
    c.store(k, v, "f32", [10, 10, 10], [65, -1, 100])  # five rows fit; none; none
    assert status(lz, device) & 2
    c.store_model(kv[:5], vv[:5], [5], [65])
    c.check()
    for starts in ([0, 10, 20, 31], [-4, 10, 20, 30]):
        before = c.read()
        c.store(k, v, "f32", None, [70, 70, 70], starts=starts)
        assert status(lz, device) & 2
        for a, b in zip(before, c.read()):
            np.testing.assert_array_equal(a, b)
    c.dispose()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,nkv,block", [(64, 2, 32), (128, 3, 128), (128, 1, 64)])
def test_load_matches_the_definition(lz, device, suite, hd, nkv, block, dt):
    rng = np.random.default_rng(hd)
    c = Cache(lz, device, suite, 4, 333, nkv, hd, block, rng)
    for n, pos in [([333, 0, 100, 7], [0, 3, 200, 326]), ([1, 1, 1, 1], [332, 0, 31, 64])]:
        rows, width = sum(n), nkv * hd
        st, po = c.int_buffer(np.concatenate([[0], np.cumsum(n)]) + 1), c.int_buffer(pos)
        stride = width + 8
        out = [lz.SharedBuffer(device, code(lz, dt), (rows + 3) * stride) for _ in range(2)]
        suite.KvCacheQ8.Load(device, *c.buffers, *out, st, po, nkv, hd, block, c.max_seq, 4, rows + 3, stride, stride)
        for w in range(2):
            got = from_type(out[w].ToArray(), dt).reshape(rows + 3, stride)
            assert np.all(got[0] == 0) and np.all(got[rows + 1:] == 0) and np.all(got[:, width:] == 0)
            want = np.concatenate([so.values(c.codes[w][i], c.scales[w][i], block)[p:p + m] for i, (m, p) in
                                   enumerate(zip(n, pos))]).reshape(rows, width)
            want = from_type(as_type(want.astype(np.float32), dt)[0], dt)  # code * scale rounded to f32, then to the type
            np.testing.assert_array_equal(got[1:rows + 1, :width], want)
        for x in (st, po, *out):
            x.Dispose()
    assert status(lz, device) == 0
    c.dispose()


@pytest.mark.parametrize("count", [1, 31, 32, 33, 64, 65, 1023, 1024, 1025])
def test_load_of_many_sequences(lz, device, suite, count):
    # empty ones among them, at both ends too, and rows in front of the first and behind the last
    rng = np.random.default_rng(count)
    c = Cache(lz, device, suite, count, 8, 1, 64, 32, rng)
    n, pos = rng.integers(0, 4, count), rng.integers(0, 5, count)
    n[0] = n[-1] = 0
    n[count // 2] = 4
    rows = int(n.sum()) + 5
    st, po = c.int_buffer(np.concatenate([[0], np.cumsum(n)]) + 3), c.int_buffer(pos)
    out = [lz.SharedBuffer.from_array(device, np.full(rows * 64, 9, np.float32)) for _ in range(2)]
    status(lz, device)
    suite.KvCacheQ8.Load(device, *c.buffers, *out, st, po, 1, 64, 32, 8, count, rows)
    assert status(lz, device) == 0
    for w in range(2):
        got = out[w].ToArray().reshape(rows, 64)
        assert np.all(got[:3] == 9) and np.all(got[rows - 2:] == 9)
        want = np.concatenate([so.values(c.codes[w][i], c.scales[w][i], 32)[p:p + m] for i, (m, p) in enumerate(zip(n, pos))])
        np.testing.assert_array_equal(got[3:rows - 2], want[:, 0].astype(np.float32))
    for x in (st, po, *out):
        x.Dispose()
    c.dispose()


def test_load_outside_the_cache(lz, device, suite):
    rng = np.random.default_rng(3)
    c = Cache(lz, device, suite, 2, 40, 1, 64, 32, rng)
    st, po = c.int_buffer([0, 10, 20]), c.int_buffer([35, -3])
    out = [lz.SharedBuffer(device, lz.F32, 20 * 64) for _ in range(2)]
    status(lz, device)
    suite.KvCacheQ8.Load(device, *c.buffers, *out, st, po, 1, 64, 32, 40, 2, 20)
    assert status(lz, device) & 2
    for w in range(2):
        got = out[w].ToArray().reshape(20, 64)
        assert np.all(got[5:] == 0)
        np.testing.assert_array_equal(got[:5], so.values(c.codes[w][0], c.scales[w][0], 32)[35:40, 0].astype(np.float32))
    for x in (st, po, *out):
        x.Dispose()
    c.dispose()


@pytest.mark.parametrize("starts", [[I32_MAX, I32_MIN], [I32_MIN, 6], [I32_MIN + 3, 6], [I32_MIN, I32_MIN], [7, 9]])
def test_starts_far_outside(lz, device, suite, starts):
    # differences that overflow, rows behind the buffer: no row that an op could serve, so all buffers stay as they are
    rng = np.random.default_rng(33)
    c = Cache(lz, device, suite, 1, 4, 1, 64, 32, rng)
    st, po = c.int_buffer(starts), c.int_buffer([0])
    x = [lz.SharedBuffer.from_array(device, np.full(6 * 64, 3, np.float32)) for _ in range(2)]
    status(lz, device)
    suite.KvCacheQ8.Load(device, *c.buffers, *x, st, po, 1, 64, 32, 4, 1, 6)
    assert status(lz, device) == 2
    suite.KvCacheQ8.Store(device, *x, *c.buffers, st, po, 1, 64, 32, 4, 1, 6)
    assert status(lz, device) == 2
    c.check()
    if starts[1] != 6:
        suite.Attention.ExecuteQ8(device, x[0], *c.buffers, x[1], st, po, 64, 1, 1, 32, 4, 1, 6)
        assert status(lz, device) == 2
    for b in x:
        assert np.all(b.ToArray() == 3)
    for b in (st, po, *x):
        b.Dispose()
    c.dispose()


# ----------------------------------------------------------------------------------------------
# Attention over the cache
# ----------------------------------------------------------------------------------------------

# f32 and f16 results: weights as sums of two f16 terms, off by 2^-21 at most. bf16 results: weights rounded once to
# f16, and a rounding is off by at most half a step, 2^-11 relative.
UNIT_P = {"f32": 2.0 ** -21, "f16": 2.0 ** -21, "bf16": 2.0 ** -11}


def attend(lz, device, suite, c, nh, n, lengths, dt, seed=0, starts="sum", gain=1.0, fill=7.0):
    """Runs ExecuteQ8; returns (got, want, bound)."""
    rng = np.random.default_rng(seed)
    rows = sum(n)
    q, qv = as_type(rng.standard_normal((rows, nh * c.hd)) * gain, dt)
    st = c.int_buffer(np.concatenate([[0], np.cumsum(n)]) if isinstance(starts, str) else starts)
    le = c.int_buffer(lengths)
    qb = lz.SharedBuffer.from_array(device, q, code(lz, dt))
    ob = lz.SharedBuffer.from_array(device, as_type(np.full((rows, nh * c.hd), fill), dt)[0], code(lz, dt))
    suite.Attention.ExecuteQ8(device, qb, *c.buffers, ob, st, le, c.hd, nh, c.nkv, c.block, c.max_seq, c.count, rows)
    got = from_type(ob.ToArray(), dt).reshape(rows, nh, c.hd)
    for x in (st, le, qb, ob):
        if x is not None:
            x.Dispose()
    want, bound = np.zeros(got.shape), np.zeros(got.shape)
    a = 0
    for i, (m, length) in enumerate(zip(n, lengths)):
        k, v = (so.values(c.codes[w][i][:length], c.scales[w][i], c.block).reshape(length, c.nkv * c.hd)
            for w in range(2))
        o, *errs = so.attention(qv[a:a + m], k, v, np.arange(length - m, length), nh, c.nkv)
        want[a:a + m], bound[a:a + m] = o, so.attention_bound(o, *errs, c.hd, UNIT_P[dt], UNIT[dt])
        a += m
    return got, want, bound


def assert_within(got, want, bound):
    err = np.abs(got - want)
    assert np.all(err <= bound), f"{np.nanmax(err / bound):.3g} of the bound, max err {np.nanmax(err):.3g}"


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,nh,nkv,block", [(128, 28, 4, 64), (64, 14, 2, 32), (128, 8, 8, 128), (64, 12, 1, 64),
                                             (128, 16, 1, 32), (64, 40, 2, 128), (128, 6, 2, 32)])
def test_decode_batch(lz, device, suite, hd, nh, nkv, block, dt):
    rng = np.random.default_rng(hd + nh)
    c = Cache(lz, device, suite, 9, 611, nkv, hd, block, rng, scale=0.01)
    lengths = [1, 31, 32, 33, 0, 127, 129, 611, 300]
    got, want, bound = attend(lz, device, suite, c, nh, [1] * 9, lengths, dt, starts=None)
    assert_within(got, want, bound)
    assert np.all(got[4] == 0)
    assert status(lz, device) == 0
    c.dispose()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("hd,nh,nkv,block", [(128, 28, 4, 64), (64, 14, 2, 32), (64, 9, 3, 128), (128, 12, 1, 32)])
def test_several_rows_a_sequence(lz, device, suite, hd, nh, nkv, block, dt):
    rng = np.random.default_rng(nh)
    c = Cache(lz, device, suite, 7, 260, nkv, hd, block, rng, scale=0.01)
    n, lengths = [1, 5, 0, 17, 2, 33, 9], [200, 5, 77, 260, 130, 33, 3]  # the last has rows that see nothing
    got, want, bound = attend(lz, device, suite, c, nh, n, lengths, dt)
    assert_within(got, want, bound)
    assert np.all(got[-9:-3] == 0)
    c.dispose()


@pytest.mark.parametrize("count,length,nh,nkv", [(1, 20000, 8, 1), (1, 9000, 28, 4), (3, 6000, 14, 2), (40, 700, 8, 8)])
def test_long_contexts(lz, device, suite, count, length, nh, nkv):
    rng = np.random.default_rng(length)
    c = Cache(lz, device, suite, count, length, nkv, 128 if nh != 14 else 64, 64, rng, scale=0.01)
    lengths = [max(1, length - 997 * i % length) for i in range(count)]
    got, want, bound = attend(lz, device, suite, c, nh, [1] * count, lengths, "f32")
    assert_within(got, want, bound)
    c.dispose()


def test_more_kv_heads_than_ctas(lz, device, suite):
    # heads take turns: 200 KV heads on one team of warps a CTA
    rng = np.random.default_rng(21)
    c = Cache(lz, device, suite, 2, 3100, 200, 64, 64, rng, scale=0.01)
    got, want, bound = attend(lz, device, suite, c, 200, [1, 1], [3100, 2900], "f32", starts=None)
    assert_within(got, want, bound)
    c.dispose()


def test_as_many_sequences_as_a_call_takes(lz, device, suite):
    rng = np.random.default_rng(22)
    count, max_seq = 4096, 40
    c = Cache(lz, device, suite, count, max_seq, 1, 128, 32)
    n = rng.integers(0, 3, count)
    n[100], pos = 30, np.zeros(count, int)
    (k, v), (kv, vv) = rows_of(rng, int(n.sum()), 128, "f16")
    c.store(k, v, "f16", n, pos)
    c.store_model(kv, vv, n, pos)
    c.check()
    got, want, bound = attend(lz, device, suite, c, 2, n.tolist(), n.tolist(), "f32")
    assert_within(got, want, bound)
    rows = int(n.sum())
    st, po = c.int_buffer(np.concatenate([[0], np.cumsum(n)])), c.int_buffer(pos)
    out = [lz.SharedBuffer(device, lz.F32, rows * 128) for _ in range(2)]
    suite.KvCacheQ8.Load(device, *c.buffers, *out, st, po, 1, 128, 32, max_seq, count, rows)
    for w in range(2):
        want = np.concatenate([so.values(c.codes[w][i, :m], c.scales[w][i], 32) for i, m in enumerate(n)])
        np.testing.assert_array_equal(out[w].ToArray().reshape(rows, 128), want[:, 0].astype(np.float32))
    for x in (st, po, *out):
        x.Dispose()
    c.dispose()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_query_that_is_not_finite_spoils_its_own_row(lz, device, suite, bad, dt):
    rng = np.random.default_rng(23)
    c = Cache(lz, device, suite, 2, 300, 2, 64, 32, rng, scale=0.01)
    q = rng.standard_normal((3, 14, 64))
    le, st = c.int_buffer([300, 77]), c.int_buffer([0, 2, 3])
    got = []
    for spoil in (False, True):
        if spoil:
            q[1, 4, 9] = bad
        with lz.SharedBuffer.from_array(device, as_type(q, dt)[0], code(lz, dt)) as qb, \
                lz.SharedBuffer(device, code(lz, dt), q.size) as ob:
            suite.Attention.ExecuteQ8(device, qb, *c.buffers, ob, st, le, 64, 14, 2, 32, 300, 2, 3)
            got.append(from_type(ob.ToArray(), dt).reshape(3, 14, 64))
    assert not np.isfinite(got[1][1, 4]).any()
    got[1][1, 4] = got[0][1, 4]
    np.testing.assert_array_equal(got[0], got[1])
    for x in (le, st):
        x.Dispose()
    c.dispose()


def test_descending_starts_run_nothing(lz, device, suite):
    rng = np.random.default_rng(24)
    c = Cache(lz, device, suite, 3, 64, 1, 64, 32, rng, scale=0.01)
    st, le = c.int_buffer([0, 6, 1, 6]), c.int_buffer([60, 60, 60])  # eleven rows out of six
    status(lz, device)
    with lz.SharedBuffer(device, lz.F32, 6 * 64) as qb, lz.SharedBuffer.from_array(device, np.full(6 * 64, 3, np.float32)) as ob:
        suite.Attention.ExecuteQ8(device, qb, *c.buffers, ob, st, le, 64, 1, 1, 32, 64, 3, 6)
        assert status(lz, device) & 2
        assert np.all(ob.ToArray() == 3)
    for x in (st, le):
        x.Dispose()
    c.dispose()


def test_scales_that_differ_much(lz, device, suite):
    # a loud block beside quiet ones: their share of the output keeps its accuracy
    rng = np.random.default_rng(5)
    c = Cache(lz, device, suite, 1, 512, 2, 64, 32, rng, scale=0.01)
    c.scales[1][0, ::3] *= 1e4
    c.scales[1][0, 1::3] *= 1e-6
    c.scales[1][0, 5] = 0
    c.scales[0][0, 7] = 0
    for b, x in zip(c.buffers[2:], c.scales):
        b.Write(x)
    got, want, bound = attend(lz, device, suite, c, 14, [3], [500], "f32")
    assert_within(got, want, bound)
    c.dispose()


@pytest.mark.parametrize("gain", [1e-6, 30.0, 3000.0])
def test_query_magnitudes(lz, device, suite, gain):
    rng = np.random.default_rng(6)
    c = Cache(lz, device, suite, 2, 200, 2, 128, 64, rng, scale=0.01)
    got, want, bound = attend(lz, device, suite, c, 14, [1, 4], [200, 150], "f32", gain=gain)
    assert_within(got, want, bound)
    c.dispose()


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_what_lies_behind_a_sequence(lz, device, suite, dt, bad):
    rng = np.random.default_rng(7)
    c = Cache(lz, device, suite, 3, 400, 2, 64, 32, rng, scale=0.01)
    n, lengths = [1, 3, 1], [37, 96, 200]
    got, want, bound = attend(lz, device, suite, c, 6, n, lengths, dt)
    assert_within(got, want, bound)
    for i, length in enumerate(lengths):
        for w in range(2):
            c.codes[w][i, length:] = 127
            c.scales[w][i, -(-length // 32):] = bad  # blocks that hold nothing yet
    for b, x in zip(c.buffers, (*c.codes, *c.scales)):
        b.Write(x)
    again, _, _ = attend(lz, device, suite, c, 6, n, lengths, dt)
    np.testing.assert_array_equal(again, got)
    c.scales[1][2, 3] = bad  # and one that is seen shows
    c.buffers[3].Write(c.scales[1])
    again, _, _ = attend(lz, device, suite, c, 6, n, lengths, dt)
    np.testing.assert_array_equal(again[:4], got[:4])
    assert not np.any(np.isfinite(again[4:, :3]) & np.isfinite(again[4:, 3:])) or np.isinf(bad)
    assert not np.all(np.isfinite(again[4:]))
    c.dispose()


def test_lengths_outside_the_cache(lz, device, suite):
    rng = np.random.default_rng(8)
    c = Cache(lz, device, suite, 3, 100, 2, 64, 32, rng, scale=0.01)
    good = attend(lz, device, suite, c, 4, [1, 1, 1], [100, 0, 50], "f32")
    assert_within(*good)
    status(lz, device)
    st, le = c.int_buffer([0, 1, 2, 3]), c.int_buffer([1 << 30, -7, 50])
    q = as_type(np.random.default_rng(0).standard_normal((3, 256)), "f32")[0]
    with lz.SharedBuffer.from_array(device, q) as qb, lz.SharedBuffer(device, lz.F32, 3 * 256) as ob:
        suite.Attention.ExecuteQ8(device, qb, *c.buffers, ob, st, le, 64, 4, 2, 32, 100, 3, 3)
        np.testing.assert_array_equal(ob.ToArray().reshape(3, 4, 64).astype(np.float64), good[0])  # cut to [0, max_seq]
        assert status(lz, device) & 2
        st.Write(np.array([0, 1, 2, 9], np.int32))
        suite.Attention.ExecuteQ8(device, qb, *c.buffers, ob, st, le, 64, 4, 2, 32, 100, 3, 3)
        assert status(lz, device) & 2
    for x in (st, le):
        x.Dispose()
    c.dispose()


def test_rows_outside_the_starts_are_left(lz, device, suite):
    rng = np.random.default_rng(9)
    c = Cache(lz, device, suite, 2, 64, 1, 64, 32, rng, scale=0.01)
    st, le = c.int_buffer([2, 3, 5]), c.int_buffer([60, 30])
    q = rng.standard_normal((8, 128)).astype(np.float32)
    with lz.SharedBuffer.from_array(device, q) as qb, lz.SharedBuffer.from_array(device, np.full((8, 128), 3, np.float32)) as ob:
        suite.Attention.ExecuteQ8(device, qb, *c.buffers, ob, st, le, 64, 2, 1, 32, 64, 2, 8)
        got = ob.ToArray().reshape(8, 128)
    assert np.all(got[:2] == 3) and np.all(got[5:] == 3) and not np.any(got[2:5] == 3)
    for x in (st, le):
        x.Dispose()
    c.dispose()


def test_strided_rows(lz, device, suite):
    rng = np.random.default_rng(10)
    c = Cache(lz, device, suite, 2, 64, 2, 64, 32, rng, scale=0.01)
    le = c.int_buffer([60, 30])
    q = rng.standard_normal((2, 8 * 64)).astype(np.float32)
    wide = np.zeros((2, 8 * 64 + 4), np.float32)
    wide[:, :512] = q
    with lz.SharedBuffer.from_array(device, q) as qb, lz.SharedBuffer.from_array(device, wide) as wb, \
            lz.SharedBuffer(device, lz.F32, 1024) as ob, lz.SharedBuffer(device, lz.F32, 2 * 520) as sb:
        suite.Attention.ExecuteQ8(device, qb, *c.buffers, ob, None, le, 64, 8, 2, 32, 64, 2, 2)
        suite.Attention.ExecuteQ8(device, wb, *c.buffers, sb, None, le, 64, 8, 2, 32, 64, 2, 2, 516, 520)
        got = sb.ToArray().reshape(2, 520)
        np.testing.assert_array_equal(got[:, :512], ob.ToArray().reshape(2, 512))
        assert np.all(got[:, 512:] == 0)
    le.Dispose()
    c.dispose()


def test_offsets_past_32_bits(lz, device, suite):
    # the second sequence's codes start behind 2^31 bytes
    max_seq, nkv, hd, block = 2_200_000, 8, 128, 128
    blocks = -(-max_seq // block)
    rng = np.random.default_rng(11)
    bufs = [lz.SharedBuffer(device, lz.I8, 2 * max_seq * nkv * hd) for _ in range(2)]
    bufs += [lz.SharedBuffer(device, lz.F32, 2 * blocks * nkv) for _ in range(2)]
    n, pos = 150, max_seq - 150
    (k, v), (kv, vv) = rows_of(rng, n, nkv * hd, "f32")
    st, po = (lz.SharedBuffer.from_array(device, np.array(x, np.int32)) for x in ([0, 0, n], [0, pos]))
    kb, vb, ko, vo = (lz.SharedBuffer.from_array(device, x) for x in (k, v, k * 0, v * 0))
    suite.KvCacheQ8.Store(device, kb, vb, *bufs, st, po, nkv, hd, block, max_seq, 2, n)
    suite.KvCacheQ8.Load(device, *bufs, ko, vo, st, po, nkv, hd, block, max_seq, 2, n)
    seen = 150
    for got, x in ((ko, kv), (vo, vv)):
        codes, scales = np.zeros((block * 3, nkv, hd), np.int8), np.zeros((3, nkv), np.float32)
        so.store(x.reshape(n, nkv, hd).astype(np.float64), codes, scales, pos % block, block)
        want = so.values(codes, scales, block)[pos % block:pos % block + n].reshape(n, -1).astype(np.float32)
        np.testing.assert_array_equal(got.ToArray().reshape(n, -1), want)
    assert seen == 150
    q = rng.standard_normal((1, nkv * hd)).astype(np.float32)
    le = lz.SharedBuffer.from_array(device, np.array([0, max_seq], np.int32))
    qs = lz.SharedBuffer.from_array(device, np.array([0, 0, 1], np.int32))
    with lz.SharedBuffer.from_array(device, q * 3) as qb, lz.SharedBuffer(device, lz.F32, nkv * hd) as ob:
        suite.Attention.ExecuteQ8(device, qb, *bufs, ob, qs, le, hd, nkv, nkv, block, max_seq, 2, 1)
        got = ob.ToArray().reshape(nkv, hd)
    # keys that were never stored score 0 with a value of 0
    kk, vvv = (b.ToArray().reshape(n, nkv, hd).astype(np.float64) for b in (ko, vo))
    s = np.einsum("jhd,hd->hj", kk, q.reshape(nkv, hd).astype(np.float64) * 3) / np.sqrt(hd)
    w = np.exp(s)
    total = w.sum(1, keepdims=True) + (max_seq - n)
    want = np.einsum("hj,jhd->hd", w / total, vvv)
    # 2^21 weights of 1 summed in f32 by splits and tiles: 2^-23 a step over at most 2^12 steps of a split
    assert np.all(np.abs(got - want) <= 2.0 ** -10 * np.abs(want).max())
    for x in (st, po, kb, vb, ko, vo, le, qs, *bufs):
        x.Dispose()


def test_same_call_gives_the_same_bits_and_lists_share_the_scratch(lz, device, suite):
    rng = np.random.default_rng(12)
    c = Cache(lz, device, suite, 4, 3000, 2, 128, 64, rng, scale=0.01)
    e = Cache(lz, device, suite, 2, 5000, 1, 64, 32, rng, scale=0.01)
    qc = lz.SharedBuffer.from_array(device, rng.standard_normal((4, 8 * 128)).astype(np.float32))
    qe = lz.SharedBuffer.from_array(device, rng.standard_normal((2, 7 * 64)).astype(np.float32))
    oc, oe = lz.SharedBuffer(device, lz.F32, 4 * 1024), lz.SharedBuffer(device, lz.F32, 2 * 448)
    lc, le = c.int_buffer([3000, 1, 777, 2050]), e.int_buffer([5000, 4097])

    def call():
        suite.Attention.ExecuteQ8(device, qc, *c.buffers, oc, None, lc, 128, 8, 2, 64, 3000, 4, 4)
        suite.Attention.ExecuteQ8(device, qe, *e.buffers, oe, None, le, 64, 7, 1, 32, 5000, 2, 2)

    call()
    first = oc.ToArray(), oe.ToArray()
    for recorded in (False, True, True, False):
        if recorded:
            device.BeginRecording()
        call()
        if recorded:
            device.EndRecording()
        np.testing.assert_array_equal(oc.ToArray(), first[0])
        np.testing.assert_array_equal(oe.ToArray(), first[1])
    # a replayed list reads the lengths of its time
    lc.Write(np.array([10, 2000, 64, 1], np.int32))
    device.BeginRecording()
    call()
    device.EndRecording()
    listed = oc.ToArray()
    call()
    np.testing.assert_array_equal(oc.ToArray(), listed)
    assert not np.array_equal(listed, first[0])
    for x in (qc, qe, oc, oe, lc, le):
        x.Dispose()
    c.dispose()
    e.dispose()


def test_refusals(lz, device, suite):
    rng = np.random.default_rng(13)
    c = Cache(lz, device, suite, 2, 100, 2, 64, 32, rng, scale=0.01)
    f = lz.SharedBuffer(device, lz.F32, 2 * 256)
    h = lz.SharedBuffer(device, lz.F16, 2 * 256)
    i = c.int_buffer([0, 1, 2])
    few = [c.buffers[0].View(0, c.buffers[0].Count - 1), c.buffers[2].View(0, c.buffers[2].Count - 1)]

    def attn(q=f, kc=c.buffers[0], ks=c.buffers[2], out=f, st=i, le=i, hd=64, nh=4, nkv=2, block=32, ms=100, count=2,
             tokens=2, strides=()):
        suite.Attention.ExecuteQ8(device, q, kc, c.buffers[1], ks, c.buffers[3], out, st, le, hd, nh, nkv, block, ms,
                                  count, tokens, *strides)

    def kv(op, k=f, v=f, kc=c.buffers[0], ks=c.buffers[2], st=i, po=i, nkv=2, hd=64, block=32, ms=100, count=2,
           tokens=2, strides=()):
        cache = (kc, c.buffers[1], ks, c.buffers[3])
        first = (k, v, *cache) if op == "Store" else (*cache, k, v)
        getattr(suite.KvCacheQ8, op)(device, *first, st, po, nkv, hd, block, ms, count, tokens, *strides)

    A, R, U = lz.ArgumentException, lz.ArgumentOutOfRangeException, lz.NotSupportedException
    before = c.read()
    shared = [(U, dict(hd=96)), (U, dict(block=48)), (R, dict(ms=0)), (R, dict(count=-1)), (R, dict(count=4097)),
              (A, dict(kc=few[0])), (A, dict(ks=few[1])), (A, dict(kc=f)), (A, dict(ks=h)), (A, dict(tokens=200)),
              (A, dict(st=None, tokens=1)), (A, dict(st=f)), (R, dict(tokens=-1)), (A, dict(strides=(5,))),
              (A, dict(strides=(257,)))]
    for error, kw in shared + [(A, dict(nh=3)), (A, dict(out=h)), (A, dict(q=c.buffers[0])), (A, dict(le=f))]:
        with pytest.raises(error):
            attn(**kw)
    for op in ("Store", "Load"):
        for error, kw in shared + [(A, dict(v=h)), (A, dict(k=c.buffers[0], v=c.buffers[0])), (A, dict(po=f))]:
            with pytest.raises(error):
                kv(op, **kw)
        kv(op, count=0, tokens=0)
    attn(count=0, tokens=0)
    for a, b in zip(before, c.read()):
        np.testing.assert_array_equal(a, b)
    for x in (f, h, i, *few):
        x.Dispose()
    c.dispose()


# ----------------------------------------------------------------------------------------------
# Together
# ----------------------------------------------------------------------------------------------

def test_prompts_stored_decoded_and_continued(lz, device, suite):
    """Prompts attended packed and stored, tokens decoded from the cache in a replayed list, then a prompt that
    continues the cached sequences: their keys loaded in front of the new ones."""
    hd, nh, nkv, block, max_seq = 64, 6, 2, 32, 160
    rng = np.random.default_rng(14)
    prompt = [70, 1, 31]
    c = Cache(lz, device, suite, 3, max_seq, nkv, hd, block)
    starts = np.concatenate([[0], np.cumsum(prompt)])
    rows = sum(prompt)
    k, v, q = (rng.standard_normal((rows, w * hd)).astype(np.float32) for w in (nkv, nkv, nh))
    bufs = {}

    def put(name, x, dt="f32"):
        bufs[name] = lz.SharedBuffer.from_array(device, as_type(x, dt)[0], code(lz, dt))
        return bufs[name]

    kb, vb, qb = put("k", k), put("v", v), put("q", q)
    k16, v16 = (bufs.setdefault(x, lz.SharedBuffer(device, lz.F16, rows * nkv * hd)) for x in ("k16", "v16"))
    ob = put("o", q * 0)
    st, zero = c.int_buffer(starts), c.int_buffer([0, 0, 0])
    suite.KvCacheStore.ExecuteRows(device, kb, vb, k16, v16, 0, nkv * hd, rows)  # the packed rows in 16 bits
    suite.Attention.ExecutePacked(device, qb, k16, v16, ob, st, None, hd, nh, nkv, 3, rows, rows)
    suite.KvCacheQ8.Store(device, kb, vb, *c.buffers, st, zero, nkv, hd, block, max_seq, 3, rows)
    got = ob.ToArray().reshape(rows, nh, hd)
    c.store_model(k, v, prompt, [0, 0, 0])
    c.check()
    for i, n in enumerate(prompt):
        a = slice(starts[i], starts[i + 1])
        kk, vv = (from_type(as_type(x[a], "f16")[0], "f16") for x in (k, v))
        o, *errs = so.attention(q[a], kk, vv, np.arange(n), nh, nkv)
        assert_within(got[a], o, so.attention_bound(o, *errs, hd, UNIT_P["f32"], UNIT["f32"]))
    # decode: the same list each step, positions and lengths written before it
    lengths = np.array(prompt, np.int32)
    po, le = c.int_buffer(lengths), c.int_buffer(lengths + 1)
    tk, tv, tq, to = (lz.SharedBuffer(device, lz.F32, 3 * w * hd) for w in (nkv, nkv, nh, nh))
    for step in range(40):
        x = [rng.standard_normal((3, w * hd)).astype(np.float32) * (1 + step / 20) for w in (nkv, nkv, nh)]
        for b, y in zip((tk, tv, tq), x):
            b.Write(y)
        po.Write(lengths)
        le.Write(lengths + 1)
        device.BeginRecording()
        suite.KvCacheQ8.Store(device, tk, tv, *c.buffers, None, po, nkv, hd, block, max_seq, 3, 3)
        suite.Attention.ExecuteQ8(device, tq, *c.buffers, to, None, le, hd, nh, nkv, block, max_seq, 3, 3)
        device.EndRecording()
        c.store_model(x[0], x[1], [1, 1, 1], lengths)
        lengths += 1
        if step % 13 == 0 or step == 39:
            c.check()
            got = to.ToArray().reshape(3, nh, hd)
            for i in range(3):
                kk, vv = (so.values(c.codes[w][i][:lengths[i]], c.scales[w][i], block).reshape(lengths[i], -1)
                          for w in range(2))
                o, *errs = so.attention(x[2][i:i + 1], kk, vv, [lengths[i] - 1], nh, nkv)
                assert_within(got[i:i + 1], o, so.attention_bound(o, *errs, hd, UNIT_P["f32"], UNIT["f32"]))
    # continue: load what is cached in front of new rows, in one packed buffer
    new = [20, 9, 33]
    total = [int(a + b) for a, b in zip(lengths, new)]
    ks = np.concatenate([[0], np.cumsum(total)])
    nk, nv, nq = (rng.standard_normal((sum(new), w * hd)).astype(np.float32) for w in (nkv, nkv, nh))
    kall, vall = (np.zeros((ks[-1], nkv * hd), np.float16) for _ in range(2))
    ns = np.concatenate([[0], np.cumsum(new)])
    for i in range(3):
        for dst, src in ((kall, nk), (vall, nv)):
            dst[ks[i] + lengths[i]:ks[i + 1]] = src[ns[i]:ns[i + 1]].astype(np.float16)
    ka, va = lz.SharedBuffer.from_array(device, kall), lz.SharedBuffer.from_array(device, vall)
    # rows of a sequence that lie behind its cached part are left: the load's own sequences end there
    for i in range(3):
        one = [c.buffers[w].View(i * max_seq * nkv * hd, max_seq * nkv * hd) for w in range(2)]
        one += [c.buffers[2 + w].View(i * c.blocks * nkv, c.blocks * nkv) for w in range(2)]
        dst = [b.View(int(ks[i]) * nkv * hd, int(lengths[i]) * nkv * hd) for b in (ka, va)]
        sti = c.int_buffer([0, lengths[i]])
        suite.KvCacheQ8.Load(device, *one, *dst, sti, zero, nkv, hd, block, max_seq, 1, int(lengths[i]))
        for x in (*one, *dst, sti):
            x.Dispose()
    qn, on = lz.SharedBuffer.from_array(device, nq), lz.SharedBuffer(device, lz.F32, nq.size)
    stn, stk = c.int_buffer(ns), c.int_buffer(ks)
    suite.Attention.ExecutePacked(device, qn, ka, va, on, stn, stk, hd, nh, nkv, 3, sum(new), int(ks[-1]))
    got = on.ToArray().reshape(sum(new), nh, hd)
    kk, vv = (b.ToArray().reshape(-1, nkv * hd).astype(np.float64) for b in (ka, va))
    for i in range(3):
        cached = so.values(c.codes[0][i][:lengths[i]], c.scales[0][i], block).reshape(lengths[i], -1)
        np.testing.assert_array_equal(kk[ks[i]:ks[i] + lengths[i]], cached.astype(np.float32).astype(np.float16))
        a, b = slice(ns[i], ns[i + 1]), slice(ks[i], ks[i + 1])
        o, *errs = so.attention(nq[a], kk[b], vv[b], np.arange(total[i] - new[i], total[i]), nh, nkv)
        assert_within(got[a], o, so.attention_bound(o, *errs, hd, UNIT_P["f32"], UNIT["f32"]))
    assert status(lz, device) == 0
    for x in (st, zero, po, le, tk, tv, tq, to, ka, va, qn, on, stn, stk, *bufs.values()):
        x.Dispose()
    c.dispose()
