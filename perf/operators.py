"""Cases of the packed prompt attention and of the int8 KV cache (store, load, attention), in their plain form and through
the kernel suite.

A case's sequences have lengths of their own, drawn from the case's `shape` number, so that a case is always the same work.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ----------------------------------------------------------------------------------------------
# Cases
# ----------------------------------------------------------------------------------------------

def listed():
    return [
        # Three short chat turns of a 0.5B model (14 query heads, 2 KV heads of 64) prefilled in one call: latency.
        dict(name="packed few f16", op="packed", hd=64, heads=14, kv_heads=2, q="f16", kv="f16", count=3, longest=77,
             prefix=0, shape=1),
        # Eight prompts of up to 512 tokens of a 7B model (28 / 4 heads of 128) with the f32 queries that RoPE leaves.
        dict(name="packed prompts f32", op="packed", hd=128, heads=28, kv_heads=4, q="f32", kv="f16", count=8,
             longest=512, prefix=0, shape=2),
        # Sixteen ragged prompts, each behind a cached prefix of its own length.
        dict(name="packed prefix bf16", op="packed", hd=128, heads=28, kv_heads=4, q="bf16", kv="bf16", count=16,
             longest=2048, prefix=1024, shape=3),
        # One long document through a 70B model's attention (64 / 8 heads of 128).
        dict(name="packed long bf16", op="packed", hd=128, heads=64, kv_heads=8, q="bf16", kv="bf16", count=1,
             longest=16384, prefix=0, shape=4),
        # One token of one chat, 0.5B model: the smallest step, latency.
        dict(name="decode one", op="attend", hd=64, heads=14, kv_heads=2, q="f32", block=32, count=1, longest=300,
             rows=1, shape=5),
        # A decode batch of 16 (7B model), contexts up to 4096.
        dict(name="decode 16", op="attend", hd=128, heads=28, kv_heads=4, q="f32", block=64, count=16, longest=4096,
             rows=1, shape=6),
        # A decode batch of 32 (70B model), long ragged contexts: what the 8-bit cache is for.
        dict(name="decode 32 long", op="attend", hd=128, heads=64, kv_heads=8, q="bf16", block=128, count=32,
             longest=32768, rows=1, shape=7),
        # Five drafted tokens of four sequences checked at once.
        dict(name="verify drafts", op="attend", hd=128, heads=28, kv_heads=4, q="f16", block=64, count=4, longest=9001,
             rows=5, shape=8),
        # The new token of each of 16 sequences, most of them into a block that is partly filled.
        dict(name="store step", op="store", hd=128, kv_heads=4, x="f32", block=64, count=16, longest=1, start=4000,
             shape=9),
        # Eight prompts stored after their prefill.
        dict(name="store prompts", op="store", hd=128, kv_heads=8, x="bf16", block=128, count=8, longest=4096, start=0,
             shape=10),
        # Two short prefixes read back.
        dict(name="load prefixes", op="load", hd=64, kv_heads=2, x="f32", block=32, count=2, longest=200, start=30,
             shape=11),
        # Eight long contexts read back as 16-bit rows for a prompt that continues them.
        dict(name="load contexts", op="load", hd=128, kv_heads=8, x="f16", block=64, count=8, longest=16384, start=0,
             shape=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["packed", "packed", "attend", "attend", "store", "load"])
    hd, block = rng.choice([64, 128]), rng.choice([32, 64, 128])
    kv_heads, group = rng.choice([(2, 7), (4, 7), (8, 8), (8, 4), (1, 8), (6, 1), (4, 12), (3, 2)])
    shape = rng.randrange(100, 1 << 30)
    if op == "packed":
        count = _log(rng, 1, 24)
        longest = _log(rng, 1, max(2, min(8192, 40000 // count)))
        kv = rng.choice(["f16", "bf16"])
        return dict(op=op, hd=hd, heads=kv_heads * group, kv_heads=kv_heads, q=rng.choice([kv, kv, "f32"]), kv=kv,
                    count=count, longest=longest, prefix=rng.choice([0, 0, _log(rng, 1, 2048)]), shape=shape)
    if op == "attend":
        count = _log(rng, 1, 48)
        longest = _log(rng, 1, max(2, min(40000, 600000 // (count * kv_heads))))
        return dict(op=op, hd=hd, heads=kv_heads * group, kv_heads=kv_heads, q=rng.choice(["f32", "f16", "bf16"]),
                    block=block, count=count, longest=longest, rows=rng.choice([1, 1, 1, 2, 3, 7, 17]), shape=shape)
    count = _log(rng, 1, 32)
    longest = _log(rng, 1, max(2, min(16384, 150000 // count)))
    return dict(op=op, hd=hd, kv_heads=kv_heads, x=rng.choice(["f32", "f16", "bf16"]), block=block, count=count,
                longest=longest, start=rng.choice([0, _log(rng, 1, 3000)]), shape=shape)


def _lengths(case):
    """(new tokens, positions held before them) of each sequence; the first sequence has the longest."""
    r = random.Random(case["shape"])
    n, before = [], []
    for i in range(case["count"]):
        longest = case["longest"]
        length = longest if i == 0 else r.randint(max(1, longest // 8), longest)
        if case["op"] == "packed":
            n.append(length)
            before.append(r.randint(case["prefix"] // 4, case["prefix"]) if case["prefix"] else 0)
        elif case["op"] == "attend":
            rows = min(case["rows"], length)
            n.append(rows)
            before.append(length - rows)
        else:
            n.append(length)
            before.append(r.randint(case["start"] // 2, case["start"]))
    return n, before


def _starts(n):
    out = [0]
    for x in n:
        out.append(out[-1] + x)
    return out


def _slots(case):
    n, before = _lengths(case)
    return max(a + b for a, b in zip(n, before)) + 7  # a cache is seldom exactly full


def work(case):
    n, before = _lengths(case)
    hd, kvd = case["hd"], case["kv_heads"] * case["hd"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] in ("packed", "attend"):
        pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(n, before))
        flops = 4 * hd * case["heads"] * pairs
        io = 2 * sum(n) * case["heads"] * hd * size[case["q"]]
        keys = sum(n) + sum(before)
        if case["op"] == "packed":
            return {"bytes": io + 2 * keys * kvd * 2, "flops": flops}
        blocks = sum(-(-(a + b) // case["block"]) for a, b in zip(n, before))
        return {"bytes": io + 2 * keys * kvd + 8 * blocks * case["kv_heads"], "flops": flops}
    block = case["block"]
    rows = sum(n)
    touched = sum(-(-(a + b) // block) - b // block for a, b in zip(n, before))
    kept = sum(b % block for b in before)
    if case["op"] == "load":
        return {"bytes": 2 * rows * kvd * (1 + size[case["x"]]) + 8 * touched * case["kv_heads"],
                "flops": 2 * rows * kvd}
    # the rows in, the codes out (the kept ones of a block in and out), then what was stored read back as f32
    store = 2 * rows * kvd * (size[case["x"]] + 1) + 4 * kept * kvd + 8 * touched * case["kv_heads"]
    load = 2 * (rows + kept) * kvd * (1 + 4) + 8 * touched * case["kv_heads"]
    return {"bytes": store + load, "flops": 10 * rows * kvd}


# ----------------------------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------------------------

def _rows(gen, rows, width, dtype):
    """Projection rows: unit variance with a few channels that stand out, as keys and values have them."""
    gain = torch.exp(0.4 * torch.randn(width, generator=gen, device="cuda"))
    return (torch.randn(rows, width, generator=gen, device="cuda") * gain).to(dtype)


def _cache(case, gen):
    """An int8 cache as earlier stores left it: codes that fill their range, scales around 0.02."""
    count, slots, kvd = case["count"], _slots(case), case["kv_heads"] * case["hd"]
    blocks = -(-slots // case["block"])
    codes = [torch.randint(-127, 128, (count, slots, kvd), generator=gen, device="cuda", dtype=torch.int8)
             for _ in range(2)]
    scales = [torch.rand(count, blocks, case["kv_heads"], generator=gen, device="cuda") * 0.02 + 0.01
              for _ in range(2)]
    return codes + scales


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, before = _lengths(case)
    kvd = case["kv_heads"] * case["hd"]
    i32 = dict(dtype=torch.int32, device="cuda")
    s = {"n": n, "before": before}
    if case["op"] == "packed":
        s["q"] = _rows(gen, sum(n), case["heads"] * case["hd"], DTYPES[case["q"]])
        s["k"] = _rows(gen, sum(n) + sum(before), kvd, DTYPES[case["kv"]])
        s["v"] = _rows(gen, sum(n) + sum(before), kvd, DTYPES[case["kv"]])
        s["q_starts"] = torch.tensor(_starts(n), **i32)
        s["kv_starts"] = torch.tensor(_starts([a + b for a, b in zip(n, before)]), **i32)
        return s
    s["kc"], s["vc"], s["ks"], s["vs"] = _cache(case, gen)
    s["starts"] = torch.tensor(_starts(n), **i32)
    if case["op"] == "attend":
        s["q"] = _rows(gen, sum(n), case["heads"] * case["hd"], DTYPES[case["q"]])
        s["lengths"] = torch.tensor([a + b for a, b in zip(n, before)], **i32)
    else:
        s["positions"] = torch.tensor(before, **i32)
    if case["op"] == "store":
        s["k"] = _rows(gen, sum(n), kvd, DTYPES[case["x"]])
        s["v"] = _rows(gen, sum(n), kvd, DTYPES[case["x"]])
        # What a reader of the stored blocks asks for: each sequence from the start of the first block touched.
        first = [b // case["block"] * case["block"] for b in before]
        s["read"] = [a + b - f for a, b, f in zip(n, before, first)]
        s["read_first"] = first
        s["read_starts"] = torch.tensor(_starts(s["read"]), **i32)
        s["read_positions"] = torch.tensor(first, **i32)
    return s


class _Memory:
    """A suite's buffer as torch sees it; freed with the last tensor that looks into it."""

    KINDS = {torch.float32: ("F32", "<f4"), torch.float16: ("F16", "<f2"), torch.bfloat16: ("BF16", "<i2"),
             torch.int8: ("I8", "|i1"), torch.int32: ("I32", "<i4")}

    def __init__(self, lz, device, shape, dtype):
        kind, code = self.KINDS[dtype]
        self.buffer = lz.SharedBuffer(device, getattr(lz, kind), math.prod(shape))
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": code, "version": 3,
                                         "data": (self.buffer.Pointer, False)}

    def tensor(self, dtype):
        return torch.as_tensor(self, device="cuda").view(dtype)

    def __del__(self):
        self.buffer.Dispose()


_handles = []


def _suite():
    """The process's device and kernel suite."""
    if not _handles:
        from l0llm_b200 import levelzero as lz

        device = lz.LevelZeroRuntime.GetDefaultDevice()
        _handles.extend([lz, device, lz.LlmKernelSuite.Create(device)])
    return _handles


def _into_buffers(s, case):
    """The inputs in buffers of the device, and buffers for the outputs."""
    lz, device, _ = _suite()
    new = {}
    if case["op"] in ("packed", "attend"):
        new["out"] = (s["q"].shape, s["q"].dtype)
    else:
        x = torch.float32 if case["op"] == "store" else DTYPES[case["x"]]
        rows = sum(s["read"] if case["op"] == "store" else s["n"])
        new["k_read"] = new["v_read"] = ((rows, case["kv_heads"] * case["hd"]), x)
    held, tensors = {}, {}
    todo = [(name, t.shape, t.dtype, t) for name, t in s.items() if isinstance(t, torch.Tensor)]
    todo += [(name, shape, dtype, None) for name, (shape, dtype) in new.items()]
    for name, shape, dtype, _ in todo:
        memory = _Memory(lz, device, shape, dtype)
        held[name], tensors[name] = memory.buffer, memory.tensor(dtype)
    device.Synchronize()
    for name, _, _, t in todo:
        if t is not None:
            tensors[name].copy_(t)
    torch.cuda.synchronize()
    return dict(s, **tensors, buffers=held)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    return _into_buffers(s, case) if own else s


# ----------------------------------------------------------------------------------------------
# The plain form
# ----------------------------------------------------------------------------------------------

def _attend_plain(q, k, v, scale):
    """q [n, heads, hd], k and v [m, kv_heads, hd] in f32: causal attention, the last query at the last key."""
    n, heads, hd = q.shape
    m, kv_heads = k.shape[:2]
    group = heads // kv_heads
    position = torch.arange(m - n, m, device=q.device)
    seen = torch.arange(m, device=q.device)[None, :] <= position[:, None]
    out = torch.empty_like(q)
    step = max(1, (1 << 31) // (group * n * m))  # KV heads at a time: 8 GB of scores at most
    for h in range(0, kv_heads, step):
        qh = q[:, h * group:(h + step) * group].reshape(n, -1, group, hd).permute(1, 2, 0, 3)
        kh, vh = (x[:, h:h + step].permute(1, 0, 2)[:, None] for x in (k, v))
        score = torch.matmul(qh, kh.transpose(-1, -2)) * scale
        score = score.masked_fill(~seen, -math.inf)
        top = score.amax(-1, keepdim=True)
        weight = torch.exp(score - torch.where(top.isfinite(), top, torch.zeros_like(top)))
        total = weight.sum(-1, keepdim=True)
        o = torch.matmul(weight, vh) / torch.where(total > 0, total, torch.ones_like(total))
        out[:, h * group:(h + step) * group] = o.permute(2, 0, 1, 3).reshape(n, -1, hd)
    return out


def _values(codes, scales, block, kv_heads):
    """codes [slots, kvd], scales [blocks, kv_heads] -> f32 [slots, kv_heads, hd]."""
    slots = codes.shape[0]
    each = scales.repeat_interleave(block, 0)[:slots]
    return codes.reshape(slots, kv_heads, -1).float() * each[..., None]


def _packed_plain(s, c):
    q, k, v = (s[x].float().reshape(s[x].shape[0], -1, c["hd"]) for x in ("q", "k", "v"))
    out, a, b = [], 0, 0
    for n, before in zip(s["n"], s["before"]):
        m = n + before
        out.append(_attend_plain(q[a:a + n], k[b:b + m], v[b:b + m], c["hd"] ** -0.5))
        a, b = a + n, b + m
    return torch.cat(out).reshape(s["q"].shape).to(s["q"].dtype)


def _attend_q8_plain(s, c):
    q = s["q"].float().reshape(s["q"].shape[0], -1, c["hd"])
    out, a = [], 0
    for i, (n, before) in enumerate(zip(s["n"], s["before"])):
        m = n + before
        blocks = -(-m // c["block"])
        k, v = (_values(s[x][i, :m], s[y][i, :blocks], c["block"], c["kv_heads"]) for x, y in (("kc", "ks"), ("vc", "vs")))
        out.append(_attend_plain(q[a:a + n], k, v, c["hd"] ** -0.5))
        a += n
    return torch.cat(out).reshape(s["q"].shape).to(s["q"].dtype)


def _codes(x, scale):
    """rint(x / scale) in 64 bits, where a quotient next to a half is told from the half."""
    fine = (scale > 0) & scale.isfinite()
    ratio = x.double() / torch.where(fine, scale, torch.ones_like(scale)).double()
    ratio = torch.where(fine, ratio, torch.zeros_like(ratio))
    return ratio.round().clamp(-127, 127)


def _store_plain(x, codes, scales, start, block, kv_heads):
    """Stores the rows x [n, kvd] at slots start.. of one sequence's codes [slots, kvd] and scales [blocks, kv_heads]."""
    n = x.shape[0]
    first, kept = start // block, start % block
    blocks = -(-(start + n) // block) - first
    hd = x.shape[1] // kv_heads
    rows = torch.zeros(blocks * block, kv_heads, hd, device=x.device)
    rows[kept:kept + n] = x.float().reshape(n, kv_heads, hd)
    rows = rows.reshape(blocks, block, kv_heads, hd)
    new = (rows.abs().amax((1, 3)).double() / 127).float()  # the quotient rounded once
    old = scales[first:first + blocks].clone()
    if kept:
        new[0] = torch.maximum(new[0], old[0])
    q = _codes(rows, new[:, None, :, None])
    if kept:
        was = codes[first * block:start].reshape(kept, kv_heads, hd).double() * old[0][:, None].double()
        q[0, :kept] = _codes(was, new[0][:, None])
    q = q.reshape(blocks * block, -1).to(torch.int8)
    end = min(codes.shape[0], (first + blocks) * block)
    codes[first * block:end] = q[:end - first * block]
    scales[first:first + blocks] = new


def _load_plain(codes, scales, first, rows, block, kv_heads, dtype):
    low = first // block
    each = _values(codes[low * block:first + rows], scales[low:-(-(first + rows) // block)], block, kv_heads)
    return each[first - low * block:].reshape(rows, -1).to(dtype)


def _store_load_plain(s, c):
    a = 0
    for i, (n, before) in enumerate(zip(s["n"], s["before"])):
        for x, codes, scales in (("k", "kc", "ks"), ("v", "vc", "vs")):
            _store_plain(s[x][a:a + n], s[codes][i], s[scales][i], before, c["block"], c["kv_heads"])
        a += n
    got = [torch.cat([_load_plain(s[codes][i], s[scales][i], f, r, c["block"], c["kv_heads"], torch.float32)
                      for i, (f, r) in enumerate(zip(s["read_first"], s["read"]))])
           for codes, scales in (("kc", "ks"), ("vc", "vs"))]
    return {"k": got[0], "v": got[1], "k_scales": s["ks"], "v_scales": s["vs"]}


def _load_all_plain(s, c):
    got = [torch.cat([_load_plain(s[codes][i], s[scales][i], b, n, c["block"], c["kv_heads"], DTYPES[c["x"]])
                      for i, (n, b) in enumerate(zip(s["n"], s["before"]))])
           for codes, scales in (("kc", "ks"), ("vc", "vs"))]
    return {"k": got[0], "v": got[1]}


# ----------------------------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------------------------

def _run_own(s, c):
    _, device, suite = _suite()
    b, hd, kv = s["buffers"], c["hd"], c["kv_heads"]
    count, op = c["count"], c["op"]
    if op == "packed":
        suite.Attention.ExecutePacked(device, b["q"], b["k"], b["v"], b["out"], b["q_starts"], b["kv_starts"], hd,
                                      c["heads"], kv, count, s["q"].shape[0], s["k"].shape[0])
        return s["out"]
    slots = s["kc"].shape[1]
    cache = (b["kc"], b["vc"], b["ks"], b["vs"])
    if op == "attend":
        # one row a sequence needs no starts
        starts = None if s["q"].shape[0] == count else b["starts"]
        suite.Attention.ExecuteQ8(device, b["q"], *cache, b["out"], starts, b["lengths"], hd, c["heads"], kv,
                                  c["block"], slots, count, s["q"].shape[0])
        return s["out"]
    rows = sum(s["n"])
    if op == "load":
        suite.KvCacheQ8.Load(device, *cache, b["k_read"], b["v_read"], b["starts"], b["positions"], kv, hd, c["block"],
                             slots, count, rows)
        return {"k": s["k_read"], "v": s["v_read"]}
    suite.KvCacheQ8.Store(device, b["k"], b["v"], *cache, None if rows == count else b["starts"], b["positions"], kv,
                          hd, c["block"], slots, count, rows)
    suite.KvCacheQ8.Load(device, *cache, b["k_read"], b["v_read"], b["read_starts"], b["read_positions"], kv, hd,
                         c["block"], slots, count, sum(s["read"]))
    return {"k": s["k_read"], "v": s["v_read"], "k_scales": s["ks"], "v_scales": s["vs"]}


def run(state):
    c = state["case"]
    if own:
        return _run_own(state, c)
    return {"packed": _packed_plain, "attend": _attend_q8_plain, "store": _store_load_plain,
            "load": _load_all_plain}[c["op"]](state, c)


# ----------------------------------------------------------------------------------------------
# The definition in 64 bits
# ----------------------------------------------------------------------------------------------

def _exact_attention(q, key_of, value_of, position, hd, group):
    """Query rows in slices: log-sum-exp over the keys up to each row's position, all in f64."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for h in range(q.shape[1]):
        k, v = key_of(h // group), value_of(h // group)
        index = torch.arange(k.shape[0], device=q.device)
        for r in range(0, q.shape[0], 4096):
            p = position[r:r + 4096]
            reach = int(p[-1]) + 1
            if reach <= 0:
                continue
            logit = (q[r:r + 4096, h].double() @ k[:reach].T) / math.sqrt(hd)
            logit[index[None, :reach] > p[:, None]] = -math.inf
            log_total = torch.logsumexp(logit, -1, keepdim=True)
            out[r:r + 4096, h] = torch.exp(logit - log_total) @ v[:reach]
    return out


def exact(case, seed):
    s, hd, kv = _inputs(case, seed), case["hd"], case["kv_heads"]
    if case["op"] in ("packed", "attend"):
        group, outs, a, b = case["heads"] // kv, [], 0, 0
        for i, (n, before) in enumerate(zip(s["n"], s["before"])):
            m = n + before
            q = s["q"][a:a + n].reshape(n, -1, hd)
            if case["op"] == "packed":
                k, v = (s[x][b:b + m].reshape(m, kv, hd) for x in ("k", "v"))
                of = [lambda h, x=x: x[:, h].double() for x in (k, v)]
            else:
                block = torch.arange(m, device="cuda") // case["block"]
                of = [lambda h, x=x, y=y: s[x][i, :m].reshape(m, kv, hd)[:, h].double() * s[y][i][block, h].double()[:, None]
                      for x, y in (("kc", "ks"), ("vc", "vs"))]
            position = torch.arange(before, m, device="cuda")
            outs.append(_exact_attention(q, of[0], of[1], position, hd, group).reshape(n, -1))
            a, b = a + n, b + m
        return torch.cat(outs)
    result = {}
    if case["op"] == "load":
        for x, codes, scales in (("k", "kc", "ks"), ("v", "vc", "vs")):
            parts = []
            for i, (n, before) in enumerate(zip(s["n"], s["before"])):
                slot = torch.arange(before, before + n, device="cuda")
                parts.append((s[codes][i, slot].reshape(n, kv, hd).double()
                              * s[scales][i][slot // case["block"]].double()[..., None]).reshape(n, -1))
            result[x] = torch.cat(parts)
        return result
    size = case["block"]
    for x, codes, scales in (("k", "kc", "ks"), ("v", "vc", "vs")):
        parts, table, a = [], s[scales].double(), 0
        for i, (n, before) in enumerate(zip(s["n"], s["before"])):
            end = before + n
            for at in range(before // size * size, end, size):
                lo, hi = max(at, before), min(at + size, end)
                rows = s[x][a + lo - before:a + hi - before].double().reshape(hi - lo, kv, hd)
                # a scale is a 32-bit number of the format: the codes are those of the number that is kept
                scale = (rows.abs().amax((0, 2)) / 127).float().double()
                held = None
                if at < lo:
                    old = s[scales][i, at // size].double()
                    scale = torch.maximum(scale, old)
                    held = s[codes][i, at:lo].reshape(lo - at, kv, hd).double() * old[:, None]
                    rows = torch.cat([held, rows])
                parts.append((torch.round(rows / scale[:, None]) * scale[:, None]).reshape(rows.shape[0], -1))
                table[i, at // size] = scale
            a += n
        result[x], result[x + "_scales"] = torch.cat(parts), table
    return result
