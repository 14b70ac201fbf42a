"""Attention.ExecutePacked against a plain 64-bit form: ragged lengths, prefixes, masks that leave a row empty, types,
strides, what masked places hold, recorded lists, bad starts and refusals."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import seq_oracle as so

pytestmark = pytest.mark.gpu

I32_MIN, I32_MAX = -2 ** 31, 2 ** 31 - 1
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step
# f32 queries: probabilities as sums of 16-bit terms, off by 2^-21 at most; 16-bit ones rounded to their type
UNIT_P = {"f32": 2.0 ** -21, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def as_type(x, dt):
    """(storage array, its values as f32)."""
    import torch

    x = np.ascontiguousarray(x, np.float32)
    if dt == "f32":
        return x, x
    t = torch.from_numpy(x).to(torch.float16 if dt == "f16" else torch.bfloat16)
    return t.view(torch.int16).numpy().view(np.uint16), t.float().numpy()


def from_type(x, dt):
    import torch

    if dt == "f32":
        return x.astype(np.float64)
    t = torch.from_numpy(np.ascontiguousarray(x).view(np.int16))
    return t.view(torch.float16 if dt == "f16" else torch.bfloat16).double().numpy()


def code(lz, dt):
    return {"f32": lz.F32, "f16": lz.F16, "bf16": lz.BF16}[dt]


class Packed:
    """Inputs of one call, run and compared."""

    def __init__(self, lz, device, suite, hd, nh, nkv, n, m, qt, kt, seed=0, lead=0, tail=0, edit=None):
        self.lz, self.device, self.suite = lz, device, suite
        self.hd, self.nh, self.nkv, self.n, self.m, self.qt, self.kt = hd, nh, nkv, n, m, qt, kt
        rng = np.random.default_rng(seed + hd + 7 * nh + sum(n))
        self.q_starts = np.concatenate([[0], np.cumsum(n)]).astype(np.int32) + lead
        self.kv_starts = np.concatenate([[0], np.cumsum(m)]).astype(np.int32)
        self.tokens, self.kv_tokens = int(self.q_starts[-1]) + tail, int(self.kv_starts[-1])
        q = rng.standard_normal((self.tokens, nh * hd))
        k, v = (rng.standard_normal((self.kv_tokens, nkv * hd)) for _ in range(2))
        if edit:
            edit(q, k, v)
        self.q, self.qv = as_type(q, qt)
        self.k, self.kv = as_type(k, kt)
        self.v, self.vv = as_type(v, kt)

    def buffers(self):
        lz, dev = self.lz, self.device
        mark = np.full(self.tokens * self.nh * self.hd, 7.0, np.float32)
        return [lz.SharedBuffer.from_array(dev, self.q, code(lz, self.qt)),
                lz.SharedBuffer.from_array(dev, self.k, code(lz, self.kt)),
                lz.SharedBuffer.from_array(dev, self.v, code(lz, self.kt)),
                lz.SharedBuffer.from_array(dev, as_type(mark, self.qt)[0], code(lz, self.qt)),
                lz.SharedBuffer.from_array(dev, self.q_starts), lz.SharedBuffer.from_array(dev, self.kv_starts)]

    def call(self, b, same=False):
        self.suite.Attention.ExecutePacked(self.device, *b[:5], None if same else b[5], self.hd, self.nh, self.nkv,
                                           len(self.n), self.tokens, self.kv_tokens)

    def read(self, b):
        return from_type(b[3].ToArray(), self.qt).reshape(self.tokens, self.nh, self.hd)

    def run(self, same=False):
        b = self.buffers()
        self.call(b, same)
        got = self.read(b)
        for x in b:
            x.Dispose()
        return got

    def want(self):
        out, spread, mass = (np.zeros((self.tokens, self.nh, self.hd)) for _ in range(3))
        dot = np.zeros((self.tokens, self.nh))
        for i, (n, m) in enumerate(zip(self.n, self.m)):
            a, b = self.q_starts[i], self.kv_starts[i]
            out[a:a + n], spread[a:a + n], dot[a:a + n], mass[a:a + n] = so.attention(
                self.qv[a:a + n], self.kv[b:b + m], self.vv[b:b + m], np.arange(m - n, m), self.nh, self.nkv)
        return out, spread, dot, mass

    def check(self, got):
        out, *errs = self.want()
        live = slice(self.q_starts[0], self.q_starts[-1])
        bound = so.attention_bound(out, *errs, self.hd, UNIT_P[self.qt], UNIT[self.qt])
        err = np.abs(got - out)[live]
        assert np.all(err <= bound[live]), f"{(err / bound[live]).max():.3g} of the bound, max err {err.max():.3g}"
        assert np.all(got[:live.start] == 7.0) and np.all(got[live.stop:] == 7.0)


TYPES = [("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")]


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("hd,nh,nkv", [(128, 28, 4), (64, 14, 2), (128, 4, 4), (64, 8, 1), (128, 8, 2)])
def test_ragged_sequences(lz, device, suite, hd, nh, nkv, qt, kt):
    n = [1, 33, 0, 129, 17, 64]
    c = Packed(lz, device, suite, hd, nh, nkv, n, n, qt, kt, lead=2, tail=3)
    # the packed rows of q and k are the same ones here but for the lead: both starts are given
    c.check(c.run())


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,m", [([1], [1]), ([127], [127]), ([128], [128]), ([129], [129]), ([257], [257]), ([1], [700]),
                                 ([5, 130], [300, 131]), ([40, 3], [7, 0]), ([200], [73]), ([0, 0], [4, 0])])
def test_lengths_and_prefixes(lz, device, suite, hd, n, m, qt, kt):
    c = Packed(lz, device, suite, hd, 4, 2, n, m, qt, kt, seed=len(n) + m[0])
    c.check(c.run())


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("nh,nkv", [(2, 2), (3, 1), (12, 4), (16, 1)])
def test_longer_sequences_and_groups(lz, device, suite, nh, nkv, qt, kt):
    c = Packed(lz, device, suite, 128, nh, nkv, [400, 150], [650, 150], qt, kt)
    c.check(c.run())


def test_without_kv_starts(lz, device, suite):
    c = Packed(lz, device, suite, 64, 4, 2, [70, 9, 1], [70, 9, 1], "f16", "f16")
    np.testing.assert_array_equal(c.run(same=True), c.run())


@pytest.mark.parametrize("qt,kt", TYPES)
def test_many_sequences(lz, device, suite, qt, kt):
    rng = np.random.default_rng(3)
    n = rng.integers(0, 6, 700).tolist()
    c = Packed(lz, device, suite, 64, 2, 1, n, n, qt, kt)
    c.check(c.run())


@pytest.mark.parametrize("qt,kt", [("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")])
def test_as_many_sequences_as_a_call_takes(lz, device, suite, qt, kt):
    n = (np.arange(4096) % 3 == 1).astype(int).tolist()
    n[7], n[4095] = 140, 3
    c = Packed(lz, device, suite, 128, 1, 1, n, n, qt, kt)
    c.check(c.run())


@pytest.mark.parametrize("qt,kt", TYPES)
def test_no_keys_at_all(lz, device, suite, qt, kt):
    c = Packed(lz, device, suite, 64, 2, 1, [5, 130], [0, 0], qt, kt)
    assert not c.run().any()


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_query_that_is_not_finite_spoils_its_own_row(lz, device, suite, bad, qt, kt):
    clean = Packed(lz, device, suite, 128, 4, 2, [140, 20], [200, 20], qt, kt)

    def edit(q, k, v):
        q[33, 128 + 7] = bad  # row 33, head 1

    dirty = Packed(lz, device, suite, 128, 4, 2, [140, 20], [200, 20], qt, kt, edit=edit)
    with np.errstate(all="ignore"):
        got, want = dirty.run(), clean.run()
    assert not np.isfinite(got[33, 1]).any()
    got[33, 1] = want[33, 1]
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("hd,m", [(128, 300), (64, 60)])
def test_a_row_whose_scores_are_all_minus_infinity(lz, device, suite, hd, m, qt, kt):
    # it sees keys, so it is not a row of zeros: exp(-inf - -inf) has no value
    def edit(q, k, v):
        q[3, :hd] = 0
        q[3, 0] = np.inf
        k[:, 0] = -1

    c = Packed(lz, device, suite, hd, 2, 1, [50], [m], qt, kt, edit=edit)
    b = c.buffers()
    c.call(b)
    got = c.read(b)
    assert np.all(np.isnan(got[3, 0])) and np.all(np.isfinite(got[3, 1]))
    assert np.all(np.isfinite(np.delete(got, 3, 0)))
    for x in b:
        x.Dispose()


@pytest.mark.parametrize("qt,kt", TYPES)
def test_large_scores_pick_one_key(lz, device, suite, qt, kt):
    def edit(q, k, v):
        q *= 30.0
        k[7] = 40.0 * np.sign(k[7])

    c = Packed(lz, device, suite, 64, 2, 2, [140], [200], qt, kt, edit=edit)
    got = c.run()
    out, *errs = c.want()
    bound = so.attention_bound(out, *errs, 64, UNIT_P[qt], UNIT[qt])
    assert np.all(np.abs(got - out) <= bound)


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_masked_places_hold_anything(lz, device, suite, hd, bad, qt, kt):
    # Keys and values behind a row (its own sequence's later ones, the neighbours' all) never reach it.
    n, m = [60, 150, 30], [60, 180, 30]
    clean = Packed(lz, device, suite, hd, 4, 2, n, m, qt, kt)

    def edit(q, k, v):
        k[:60], v[:60], k[240:], v[240:] = bad, bad, bad, bad  # the neighbours
        k[60 + 100:240:7] = bad                               # later keys of the sequence: rows below 70 do not see them
        v[60 + 103:240:5] = bad

    dirty = Packed(lz, device, suite, hd, 4, 2, n, m, qt, kt, edit=edit)
    with np.errstate(all="ignore"):
        got = dirty.run()
    np.testing.assert_array_equal(got[60:60 + 70], clean.run()[60:60 + 70])
    assert not np.any(np.isfinite(got[60 + 80:210]))  # a key or value that is seen shows (rows 73 on see v[163])


@pytest.mark.parametrize("qt,kt", TYPES)
def test_infinite_value_that_is_seen(lz, device, suite, qt, kt):
    def edit(q, k, v):
        v[50, 3] = np.inf
        v[70, 64 + 5] = -np.inf

    c = Packed(lz, device, suite, 64, 4, 2, [130], [130], qt, kt, edit=edit)
    with np.errstate(all="ignore"):
        got = c.run()
    finite = np.isfinite(got)
    want = np.ones_like(finite)
    want[50:, :2, 3] = False
    want[70:, 2:, 5] = False
    np.testing.assert_array_equal(finite, want)
    if qt != "f32":  # the terms of an f32 path's probabilities have both signs: an infinity shows as one or as NaN
        assert np.all(got[50:, :2, 3] == np.inf) and np.all(got[70:, 2:, 5] == -np.inf)


@pytest.mark.parametrize("qt,kt", [("f16", "f16"), ("bf16", "bf16")])
def test_views_of_a_stacked_projection(lz, device, suite, qt, kt):
    hd, nh, nkv, n = 64, 6, 2, [90, 41]
    c = Packed(lz, device, suite, hd, nh, nkv, n, n, qt, kt)
    width = (nh + 2 * nkv) * hd
    stacked = np.concatenate([c.q, c.k, c.v], 1)
    rows = stacked.shape[0]
    with lz.SharedBuffer.from_array(device, stacked, code(lz, qt)) as s, lz.SharedBuffer.from_array(device, c.q_starts) as st, \
            lz.SharedBuffer(device, code(lz, qt), rows * (nh * hd + 8)) as out:
        parts = [s.View(o, rows * width - o) for o in (0, nh * hd, (nh + nkv) * hd)]
        suite.Attention.ExecutePacked(device, *parts, out, st, None, hd, nh, nkv, len(n), rows, rows, width, width, width,
                                      nh * hd + 8)
        got = from_type(out.ToArray(), qt).reshape(rows, nh * hd + 8)
        for p in parts:
            p.Dispose()
    assert np.all(got[:, nh * hd:] == 0)  # the gap between rows is not written
    np.testing.assert_array_equal(got[:, :nh * hd].reshape(rows, nh, hd), c.run(same=True))


def test_recorded_list_follows_the_starts(lz, device, suite):
    # Two calls in one list, replayed after the starts changed: the lengths are read when the list runs.
    c = Packed(lz, device, suite, 128, 4, 2, [100, 60], [100, 60], "f16", "f16")
    e = Packed(lz, device, suite, 64, 4, 2, [33, 200], [40, 222], "f32", "f16")
    bc, be = c.buffers(), e.buffers()
    c.call(bc)
    e.call(be)  # once outside a recording
    for step in range(3):
        if step == 2:
            c.n = c.m = [30, 130]
            c.q_starts[1] = c.kv_starts[1] = 30
            bc[4].Write(c.q_starts)
            bc[5].Write(c.kv_starts)
        device.BeginRecording()
        c.call(bc)
        e.call(be)
        device.EndRecording()
        c.check(c.read(bc))
        e.check(e.read(be))
    for x in bc + be:
        x.Dispose()


@pytest.mark.parametrize("qt,kt", TYPES)
def test_same_call_gives_the_same_bits(lz, device, suite, qt, kt):
    c = Packed(lz, device, suite, 128, 8, 2, [300, 211], [300, 400], qt, kt)
    b = c.buffers()
    c.call(b)
    first = b[3].ToArray()
    for _ in range(3):
        c.call(b)
        np.testing.assert_array_equal(b[3].ToArray(), first)
    for x in b:
        x.Dispose()


def status(lz, device):
    v = C.c_int32()
    lz.check(lz.load_library().l0b_device_error_status(device.handle, C.byref(v)))
    return v.value


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("q_starts,kv_starts", [([0, 40, 500], [0, 40, 80]), ([0, 40, 80], [0, 40, 900]),
                                                ([-5, 40, 80], [0, 40, 80]), ([0, 40, 80], [-9, 40, 80])])
def test_starts_outside_the_buffers(lz, device, suite, q_starts, kv_starts, qt, kt):
    c = Packed(lz, device, suite, 64, 2, 2, [40, 40], [40, 40], qt, kt)
    status(lz, device)
    b = c.buffers()
    b[4].Write(np.array(q_starts, np.int32))
    b[5].Write(np.array(kv_starts, np.int32))
    c.call(b)
    assert status(lz, device) & 2
    b[4].Write(c.q_starts)
    b[5].Write(c.kv_starts)
    c.call(b)
    c.check(c.read(b))
    assert status(lz, device) == 0
    for x in b:
        x.Dispose()


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("q_starts,kv_starts,want", [([I32_MAX, I32_MIN], [0, 50], 7.0), ([0, 40], [1, I32_MIN], 0.0),
                                                     ([0, 40], [I32_MAX, I32_MIN], 0.0), ([I32_MIN, I32_MIN], [0, 50], 7.0)])
def test_starts_whose_differences_overflow(lz, device, suite, q_starts, kv_starts, want, qt, kt):
    # no rows at all, or rows without keys
    c = Packed(lz, device, suite, 128, 4, 2, [40], [50], qt, kt)
    b = c.buffers()
    status(lz, device)
    b[4].Write(np.array(q_starts, np.int32))
    b[5].Write(np.array(kv_starts, np.int32))
    c.call(b)
    assert status(lz, device) == 2
    np.testing.assert_array_equal(c.read(b), want)
    for x in b:
        x.Dispose()


def test_refusals(lz, device, suite):
    c = Packed(lz, device, suite, 64, 4, 2, [20, 12], [20, 12], "f16", "f16")
    b = c.buffers()

    def call(q=b[0], k=b[1], v=b[2], out=b[3], qs=b[4], ks=b[5], hd=64, nh=4, nkv=2, count=2, tokens=32, kvt=32, strides=()):
        suite.Attention.ExecutePacked(device, q, k, v, out, qs, ks, hd, nh, nkv, count, tokens, kvt, *strides)

    f32 = lz.SharedBuffer(device, lz.F32, 32 * 256)
    short = b[3].View(0, 32 * 256 - 1)
    odd = b[1].View(1, 31 * 128)
    for error, kw in [(lz.ArgumentException, dict(nh=3)), (lz.NotSupportedException, dict(hd=96)),
                      (lz.ArgumentException, dict(out=f32)), (lz.ArgumentException, dict(k=f32, v=f32)),
                      (lz.ArgumentException, dict(out=short)), (lz.ArgumentException, dict(tokens=33)),
                      (lz.ArgumentException, dict(kvt=33)), (lz.ArgumentException, dict(k=odd, kvt=30)),
                      (lz.ArgumentException, dict(strides=(255,))), (lz.ArgumentException, dict(strides=(257,))),
                      (lz.ArgumentOutOfRangeException, dict(count=-1)), (lz.ArgumentOutOfRangeException, dict(count=4097)),
                      (lz.ArgumentException, dict(count=3)), (lz.ArgumentException, dict(ks=None, kvt=31)),
                      (lz.ArgumentException, dict(qs=f32)), (lz.ArgumentOutOfRangeException, dict(tokens=-1)),
                      (lz.ArgumentOutOfRangeException, dict(strides=(1 << 62,)))]:
        with pytest.raises(error):
            call(**kw)
    call(count=0)
    call(tokens=0)
    got = from_type(b[3].ToArray(), "f16")
    assert np.all(got == 7.0)  # nothing ran
    call()
    c.check(c.read(b))
    for x in (short, odd, f32, *b):
        x.Dispose()
