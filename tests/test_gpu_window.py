"""WindowAttention on the GPU against its formulas in 64 bits.

Tolerances, with U = 2^-24 and T half a step of the tensors' type relative to
the value. A score errs by e_s = scale (D + 2) U sum |q| |k| + 4 U |s| (sums of
D products in any order; the scale, log2 e and the reference point), so a
probability by a share of e = 2 e_s + 4 U (2^x to one step). Summed over the n
keys that a row sees, with E = sum P |v|, the output errs by
  (2 max e + (n + 16) U + R) E + R' + T |out|,
R the rounding of a probability to the type (f16 2^-11, f32 0), R' what f16
loses below its normal range, n 2^-31 max |v|. lse errs by max e + (n + 16) U
and 4 steps. The way back: with W = |dout| |v| summed and A_j = W_j + sum |dout
out|, ds errs by P ((e + (D + 4) U + R) A + R sum |dout| |out|) (out itself
is rounded to the type), dq and dk sum these times |k| and |q| with n U more,
dv sums P |dout| (e + R + n U); a score's e there has lse's error too.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
T = {"f32": 2.0 ** -24, "f16": 2.0 ** -11}
SMALL = {"f32": 0.0, "f16": 2.0 ** -25}


@pytest.fixture(scope="module")
def dev():
    import torch

    from afhip import device

    device.open_device(0)
    return torch.device("cuda", 0)


def f64(x):
    return x.double().cpu().numpy()


def ints(values, dev):
    import torch

    return None if values is None else torch.tensor(values, dtype=torch.int32, device=dev)


def visible(nq, nk, left, right, sinks):
    p = np.arange(nk - nq, nk)[:, None]
    j = np.arange(nk)[None]
    seen = np.ones((nq, nk), bool)
    if right is not None:
        seen &= j <= p + right
    if left is not None:
        seen &= (j >= p - left) | (j < sinks)
    return seen


class Sequence:
    """One batch entry in 64 bits: everything for each query head."""

    def __init__(self, q, k, v, nq, nk, left, right, sinks, scale, dtype, out=None, lse=None, dout=None):
        group, d = q.shape[1] // k.shape[1], q.shape[2]
        self.out, self.out_tol = np.zeros(q.shape), np.zeros(q.shape)
        self.lse, self.lse_tol = np.full(q.shape[:2], -np.inf), np.zeros(q.shape[:2])
        self.dq, self.dk, self.dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
        self.dq_tol, self.dk_tol, self.dv_tol = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
        if nq == 0 or nk == 0:
            return
        seen = visible(nq, nk, left, right, sinks)
        some = seen.any(1)
        t = T[dtype]
        round_ = 0.0 if dtype == "f32" else t
        n = seen.sum(1)[:, None]
        for h in range(q.shape[1]):
            a, c, e = q[:nq, h], k[:nk, h // group], v[:nk, h // group]
            # What is not seen does not count, infinities and NaN neither.
            c, e = (np.where(seen.any(0)[:, None], x, 0) for x in (c, e))
            with np.errstate(invalid="ignore"):
                s = np.where(seen, a @ c.T * scale, -np.inf)
            err = np.where(seen, scale * (d + 2) * U * (np.abs(a) @ np.abs(c).T) + 4 * U * np.abs(np.where(seen, s, 0)), 0)
            share = 2 * err + 4 * U
            worst = share.max(1, keepdims=True)
            top = np.where(some[:, None], s.max(1, keepdims=True), 0)
            p = np.exp(s - top)
            total = p.sum(1, keepdims=True)
            p = p / np.where(total == 0, 1, total)
            y = p @ e
            big = np.abs(e).max()
            self.out[:nq, h] = y
            self.out_tol[:nq, h] = np.where(some[:, None], (2 * worst + (n + 16) * U + round_) * (p @ np.abs(e))
                                            + (n * 2.0 ** -31 * big if dtype == "f16" else 0) + t * np.abs(y) + SMALL[dtype], 0)
            with np.errstate(divide="ignore"):
                lse = (top + np.log(total))[:, 0]
            self.lse[:nq, h] = lse
            self.lse_tol[:nq, h] = np.where(some, worst[:, 0] + (n[:, 0] + 16) * U + 4 * 2 * U * np.abs(np.where(some, lse, 0)), 0)
            if dout is None:
                continue
            g = dout[:nq, h]
            dp, dpa = g @ e.T, np.abs(g) @ np.abs(e).T
            delta, da = (g * y).sum(1, keepdims=True), (np.abs(g) * np.abs(y)).sum(1, keepdims=True)
            share = share + 2 * np.where(some, self.lse_tol[:nq, h], 0)[:, None]
            ds = p * (dp - delta)
            ds_err = p * ((share + (d + 4) * U + round_) * (dpa + da) + t * da
                          + (np.abs(g) * self.out_tol[:nq, h]).sum(1, keepdims=True))
            # f16: ds times a power of two that keeps the largest in [2^7, 2^15]; p times 2^13.
            if dtype == "f16":
                ds_err = ds_err + 2.0 ** -32 * np.abs(ds).max()
            p_err = p * (share + round_) + (2.0 ** -38 if dtype == "f16" else 0)
            self.dq[:nq, h] = scale * ds @ c
            self.dq_tol[:nq, h] = scale * (ds_err + (nk + 8) * U * np.abs(ds)) @ np.abs(c)
            self.dk[:nk, h // group] += scale * ds.T @ a
            self.dk_tol[:nk, h // group] += scale * (ds_err + (nq * group + 8) * U * np.abs(ds)).T @ np.abs(a)
            self.dv[:nk, h // group] += p.T @ g
            self.dv_tol[:nk, h // group] += (p_err + (nq * group + 8) * U * p).T @ np.abs(g)
        for name in ("dq", "dk", "dv"):
            x, tol = getattr(self, name), getattr(self, name + "_tol")
            tol[...] = np.where(tol > 0, tol + t * np.abs(x) + SMALL[dtype], 0)


def holds(got, want, tolerance, what):
    got = f64(got)
    same = got == want  # -inf, and zeros that have to be zeros
    with np.errstate(invalid="ignore"):
        off = np.where(same, 0, np.abs(got - want))
    assert not np.isnan(off).any(), (what, "nan at", np.argwhere(np.isnan(off))[:4].tolist())
    bad = off > tolerance
    assert not bad.any(), (what, "at", np.argwhere(bad)[0].tolist(), float(off[bad].max()),
                           float((off / np.maximum(tolerance, 1e-300))[bad].max()))


def normal(rng, dev, dt, *shape, scale=1.0):
    import torch

    return torch.from_numpy((rng.normal(0, scale, shape)).astype(np.float32)).to(dev).to(dt)


def torch_dtype(dtype):
    import torch

    return torch.float16 if dtype == "f16" else torch.float32


def compare(op, q, k, v, ql, kl, dtype, dev, left, right, sinks, backward=True, seed=0, what=""):
    """One call, and the way back, against the formulas; the same bits again."""
    import torch

    b, tq, tk = q.shape[0], q.shape[1], k.shape[1]
    qi, ki = ints(ql, dev), ints(kl, dev)
    out, lse = op(q, k, v, query_lengths=qi, key_lengths=ki, return_lse=True)
    again = op(q, k, v, query_lengths=qi, key_lengths=ki)
    assert torch.equal(out, again)
    dout = None
    if backward:
        dout = normal(np.random.default_rng(seed + 100), dev, q.dtype, *q.shape)
        grads = op.backward(q, k, v, out, lse, dout, query_lengths=qi, key_lengths=ki)
        twice = op.backward(q, k, v, out, lse, dout, query_lengths=qi, key_lengths=ki)
        assert all(torch.equal(x, y) for x, y in zip(grads, twice))
    for i in range(b):
        nq, nk = tq if ql is None else min(max(ql[i], 0), tq), tk if kl is None else min(max(kl[i], 0), tk)
        s = Sequence(f64(q[i]), f64(k[i]), f64(v[i]), nq, nk, left, right, sinks, op.scale, dtype,
                     dout=None if dout is None else f64(dout[i]))
        holds(out[i], s.out, s.out_tol, (what, i, "out"))
        holds(lse[i].T, s.lse, s.lse_tol, (what, i, "lse"))
        if backward:
            for name, x in zip(("dq", "dk", "dv"), grads):
                holds(x[i], getattr(s, name), getattr(s, name + "_tol"), (what, i, name))
    return out, lse


# batch, queries, keys, query heads, key heads, head_dim, left, right, sinks, query lengths, key lengths
CASES = [
    (1, 1, 1, 1, 1, 8, None, 0, 0, None, None),
    (2, 1, 70, 4, 2, 64, 8, 0, 2, None, [70, 5]),             # steps: one window past a sink, one shorter than it
    (3, 1, 33, 8, 1, 128, None, 0, 0, [1, 0, 1], [33, 20, 0]),  # a sequence without a query, one without keys
    (1, 2, 40, 3, 3, 40, 0, 0, 0, None, None),                # each sees itself
    (2, 3, 90, 6, 2, 80, 20, None, 5, [3, 2], [90, 40]),
    (1, 33, 33, 3, 1, 32, 4, 4, 1, None, None),               # groups of 3 across a tile's end
    (2, 129, 129, 2, 2, 64, None, 0, 0, [129, 77], [129, 77]),
    (1, 200, 200, 4, 2, 128, 30, 0, 70, None, None),          # more sinks than a block of keys
    (1, 257, 300, 2, 1, 16, 64, 64, 3, None, None),
    (2, 100, 64, 2, 1, 32, None, 0, 0, None, None),           # more queries than keys: the first see nothing
    (2, 100, 64, 2, 1, 64, 10, 0, 3, [90, 100], [64, 10]),    # and the first few of those that do not see only sinks
    (1, 150, 150, 2, 2, 24, None, None, 0, [130], [140]),     # no mask but the lengths
    (1, 64, 500, 16, 2, 64, 100, 0, 4, None, None),           # a piece of a prompt
    (1, 40, 40, 2, 2, 64, 3, 0, 100, None, None),             # sinks past the last key
    (2, 31, 95, 4, 4, 128, 1000, 1000, 0, [0, 31], [95, 64]),  # windows past both ends
    (1, 130, 130, 66, 1, 32, 40, 0, 2, None, None),           # one key head for 66
    (2, 350, 350, 6, 2, 64, None, 0, 0, [350, 200], [350, 200]),  # groups of 3, the rows of a key in chunks
    (1, 400, 400, 3, 1, 128, 50, 5, 300, None, None),         # sinks over some tiles of keys
    (1, 300, 420, 2, 1, 32, 40, None, 0, None, None),         # all that follow
    (1, 300, 420, 2, 1, 128, None, 30, 0, [290], [410]),      # all that came before
]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("head_dim", [32, 64, 128])
def test_first_call_in_a_capture(head_dim, dtype, dev):
    # Nothing has run these kernels before, in this file's order: what they set up once does not disturb a capture.
    import torch

    from afhip import window

    rng, dt = np.random.default_rng(21), torch_dtype(dtype)
    op = window.WindowAttention(4, 2, head_dim, left=60, sinks=2, dtype=dtype)
    q, k, v, dout = (normal(rng, dev, dt, 1, 150, h, head_dim) for h in (4, 2, 2, 4))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = op(q, k, v, return_lse=True)
        grads = op.backward(q, k, v, out, lse, dout)
    for _ in range(3):
        for x in (q, k, v, dout):
            x.copy_(normal(rng, dev, dt, *x.shape))
        graph.replay()
        torch.cuda.synchronize()
        want, want_lse = op(q, k, v, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        assert all(torch.equal(x, y) for x, y in zip(grads, op.backward(q, k, v, want, want_lse, dout)))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_the_formulas(case, dtype, dev):
    from afhip import window

    b, tq, tk, h, hk, d, left, right, sinks, ql, kl = case
    print("window", dtype, case, flush=True)
    rng = np.random.default_rng(17)
    dt = torch_dtype(dtype)
    op = window.WindowAttention(h, hk, d, left=left, right=right, sinks=sinks, dtype=dtype)
    q, k, v = normal(rng, dev, dt, b, tq, h, d), normal(rng, dev, dt, b, tk, hk, d), normal(rng, dev, dt, b, tk, hk, d)
    compare(op, q, k, v, ql, kl, dtype, dev, left, right, sinks, what=case)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("shape", [(1, 1, 5000, 8, 2, 128), (2, 4, 3001, 4, 1, 64), (1, 100, 4000, 4, 2, 32),
                                   (1, 1, 9000, 40, 1, 64)], ids=str)
def test_split_keys(shape, dtype, dev):
    # Few rows over many keys: the parts are joined. One sequence of the second is empty.
    from afhip import window

    b, tq, tk, h, hk, d = shape
    print("window split", dtype, shape, flush=True)
    dt, rng = torch_dtype(dtype), np.random.default_rng(5)
    op = window.WindowAttention(h, hk, d, dtype=dtype)
    q, k, v = normal(rng, dev, dt, b, tq, h, d), normal(rng, dev, dt, b, tk, hk, d), normal(rng, dev, dt, b, tk, hk, d)
    compare(op, q, k, v, None, None if b == 1 else [tk - 7, 0], dtype, dev, None, 0, 0, backward=False, what=shape)
    # So short that most parts have no block.
    compare(op, q, k, v, None, [min(tk, 37)] * b, dtype, dev, None, 0, 0, backward=False, what=("short", shape))


def sampled(op, q, k, v, ql, kl, dtype, dev, left, right, sinks, pairs, backward=True, what=""):
    """A large call, and the way back, at some sequences' key heads against the formulas; the same bits again."""
    import torch

    qi, ki = ints(ql, dev), ints(kl, dev)
    out, lse = op(q, k, v, query_lengths=qi, key_lengths=ki, return_lse=True)
    assert torch.equal(out, op(q, k, v, query_lengths=qi, key_lengths=ki))
    dout = grads = None
    if backward:
        dout = normal(np.random.default_rng(99), dev, q.dtype, *q.shape)
        grads = op.backward(q, k, v, out, lse, dout, query_lengths=qi, key_lengths=ki)
        twice = op.backward(q, k, v, out, lse, dout, query_lengths=qi, key_lengths=ki)
        assert all(torch.equal(x, y) for x, y in zip(grads, twice))
    group = q.shape[2] // k.shape[2]
    for i, kv in pairs:
        heads, one = slice(kv * group, (kv + 1) * group), slice(kv, kv + 1)
        s = Sequence(f64(q[i, :, heads]), f64(k[i, :, one]), f64(v[i, :, one]), q.shape[1] if ql is None else ql[i],
                     k.shape[1] if kl is None else kl[i], left, right, sinks, op.scale, dtype,
                     dout=None if dout is None else f64(dout[i, :, heads]))
        holds(out[i, :, heads], s.out, s.out_tol, (what, i, kv, "out"))
        holds(lse[i, heads].T, s.lse, s.lse_tol, (what, i, kv, "lse"))
        if backward:
            for name, x, part in zip(("dq", "dk", "dv"), grads, (heads, one, one)):
                holds(x[i, :, part], getattr(s, name), getattr(s, name + "_tol"), (what, i, kv, name))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("head_dim", [32, 64, 128])
@pytest.mark.parametrize("batch, group", [(8, 1), (32, 1), (32, 2)])
def test_many_tiles(batch, group, head_dim, dtype, dev):
    # 128, 512 and 1,024 tiles of 128 rows: where there are many, a workgroup has fewer waves.
    from afhip import window

    print("window tiles", dtype, batch, group, head_dim, flush=True)
    rng, dt = np.random.default_rng(18), torch_dtype(dtype)
    mask = dict(left=None, right=0, sinks=0) if group == 1 else dict(left=50, right=7, sinks=3)
    op = window.WindowAttention(8 * group, 8, head_dim, dtype=dtype, **mask)
    q = normal(rng, dev, dt, batch, 200, 8 * group, head_dim)
    k, v = (normal(rng, dev, dt, batch, 230, 8, head_dim) for _ in range(2))
    ql, kl = [200 - 7 * i % 90 for i in range(batch)], [230 - 11 * i % 120 for i in range(batch)]
    pairs = [(0, 0), (batch // 2, 5), (batch - 1, 7)]
    sampled(op, q, k, v, ql, kl, dtype, dev, *mask.values(), pairs, what=(batch, group, head_dim))


@pytest.mark.parametrize("dtype, head_dim, batch", [("f16", 32, 8), ("f16", 64, 8), ("f16", 128, 2), ("f32", 32, 32),
                                                    ("f32", 64, 8), ("f32", 128, 8)])
def test_split_keys_of_many_rows(dtype, head_dim, batch, dev):
    from afhip import window

    print("window split rows", dtype, head_dim, batch, flush=True)
    rng, dt = np.random.default_rng(19), torch_dtype(dtype)
    op = window.WindowAttention(8, 8, head_dim, left=1300, sinks=40, dtype=dtype)
    q = normal(rng, dev, dt, batch, 100, 8, head_dim)
    k, v = (normal(rng, dev, dt, batch, 1500, 8, head_dim) for _ in range(2))
    ql, kl = [100, 0] + [100 - 3 * i for i in range(2, batch)], [1500, 700] + [1500 - 45 * i for i in range(2, batch)]
    pairs = [(0, 0), (1, 3), (batch - 1, 7)]
    sampled(op, q, k, v, ql, kl, dtype, dev, 1300, 0, 40, pairs, backward=False, what=(dtype, head_dim))


def test_f32_keeps_its_range(dev):
    # Values of 2^-100 and 2^100, queries and keys of 2^60 and 2^-60: three bf16 of each hold all their bits.
    from afhip import window

    rng = np.random.default_rng(20)
    op = window.WindowAttention(2, 1, 64, left=70, dtype="f32")
    for sizes in ((0, 0, -100), (0, 0, 100), (60, -60, 0), (-60, 60, -40)):
        q, k, v = (normal(rng, dev, torch_dtype("f32"), 1, 150, h, 64, scale=2.0 ** n)
                   for h, n in zip((2, 1, 1), sizes))
        compare(op, q, k, v, None, None, "f32", dev, 70, 0, 0, what=sizes)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_a_nan_stays_in_its_sequence_and_head(dtype, dev):
    import torch

    from afhip import window

    rng, dt = np.random.default_rng(22), torch_dtype(dtype)
    for tq, tk in ((150, 200), (1, 4000)):
        op = window.WindowAttention(4, 2, 64, dtype=dtype)
        q, k, v = (normal(rng, dev, dt, 2, n, h, 64) for n, h in ((tq, 4), (tk, 2), (tk, 2)))
        dout = normal(rng, dev, dt, 2, tq, 4, 64)
        want, want_lse = op(q, k, v, return_lse=True)
        grads = op.backward(q, k, v, want, want_lse, dout)
        v[1, 5, 1], k[1, 7, 1] = math.nan, math.inf
        out, lse = op(q, k, v, return_lse=True)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1, :, :2], want[1, :, :2])
        assert torch.isnan(out[1, :, 2:]).all() if tq == 1 else torch.isnan(out[1, -1, 2:]).all()
        for x, y, heads in zip(op.backward(q, k, v, out, lse, dout), grads, (2, 1, 1)):
            assert torch.equal(x[0], y[0]) and torch.equal(x[1, :, :heads], y[1, :, :heads])


def test_two_streams_at_once(dev):
    import torch

    from afhip import window

    rng, dt = np.random.default_rng(23), torch.float16
    op = window.WindowAttention(8, 2, 128, dtype="f16")
    calls = [[normal(rng, dev, dt, 1, n, h, 128) for n, h in ((80, 8), (5000, 2), (5000, 2), (80, 8))]
             for _ in range(2)]

    def run(q, k, v, dout):
        out, lse = op(q, k, v, return_lse=True)
        return out, lse, *op.backward(q, k, v, out, lse, dout)

    want = [run(*x) for x in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for n, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[n].append(run(*calls[n]))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for x in a:
            assert all(torch.equal(s, t) for s, t in zip(x, b))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_what_is_not_seen_may_hold_anything(dtype, dev):
    # Past the lengths, before every window of the call, and between the sinks and the window: infinities and NaN.
    from afhip import window

    dt, rng = torch_dtype(dtype), np.random.default_rng(6)
    for tq, h in ((1, 4), (70, 2)):
        op = window.WindowAttention(h, 2, 64, left=20, right=0, sinks=3, dtype=dtype)
        q, k, v = (normal(rng, dev, dt, 2, n, heads, 64) for n, heads in ((tq, h), (400, 2), (400, 2)))
        for x in (k, v):
            x[0, 350:], x[1, 390:] = math.nan, math.inf
            for i, n in enumerate((350, 390)):
                x[i, 3:n - tq - 20 + 0] = -math.inf if i else math.nan
        compare(op, q, k, v, None, [350, 390], dtype, dev, 20, 0, 3, what=("unseen", tq))
        q2 = q.clone()
        if tq > 1:
            q2[0, 50:] = math.nan
            compare(op, q2, k, v, [50, 70], [350, 390], dtype, dev, 20, 0, 3, backward=False, what=("rows", tq))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_what_lies_past_the_lengths_on_the_way_back(dtype, dev):
    # out, its gradient and q hold NaN past the queries, k and v past the keys: the same bits as with zeros there.
    import torch

    from afhip import window

    rng, dt = np.random.default_rng(24), torch_dtype(dtype)
    for mask in (dict(left=30, sinks=2), dict(), dict(left=5, right=9)):
        op = window.WindowAttention(4, 2, 64, dtype=dtype, **mask)
        q, dout = (normal(rng, dev, dt, 2, 100, 4, 64) for _ in range(2))
        k, v = (normal(rng, dev, dt, 2, 130, 2, 64) for _ in range(2))
        ql, kl = ints([70, 100], dev), ints([130, 90], dev)
        out, lse = op(q, k, v, query_lengths=ql, key_lengths=kl, return_lse=True)
        want = op.backward(q, k, v, out, lse, dout, query_lengths=ql, key_lengths=kl)
        for x in (q, dout, out):
            x[0, 70:] = math.nan
        for x in (k, v):
            x[1, 90:] = math.nan
        got = op.backward(q, k, v, out, lse, dout, query_lengths=ql, key_lengths=kl)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), mask


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_lengths_past_the_ends(dtype, dev):
    # Below zero and past the tensors' ends they count as the nearer end.
    import torch

    from afhip import window

    rng, dt = np.random.default_rng(25), torch_dtype(dtype)
    op = window.WindowAttention(4, 2, 32, left=30, dtype=dtype)
    q, dout = (normal(rng, dev, dt, 3, 60, 4, 32) for _ in range(2))
    k, v = (normal(rng, dev, dt, 3, 80, 2, 32) for _ in range(2))

    def both(ql, kl):
        at = dict(query_lengths=ints(ql, dev), key_lengths=ints(kl, dev))
        out, lse = op(q, k, v, return_lse=True, **at)
        return out, lse, *op.backward(q, k, v, out, lse, dout, **at)

    for a, b in zip(both([60, 0, 60], [80, 80, 0]), both([2 ** 31 - 1, -5, 61], [81, 2 ** 31 - 1, -2 ** 31])):
        assert torch.equal(a, b)


def test_f16_backward_of_large_scores(dev):
    # Scores of +-60 and gradients that grow along the keys: ds' power of two falls again and again.
    import torch

    from afhip import window

    rng, dt = np.random.default_rng(26), torch_dtype("f16")
    op = window.WindowAttention(4, 2, 64, right=None, dtype="f16")
    q, k = normal(rng, dev, dt, 1, 90, 4, 64, scale=4.0), normal(rng, dev, dt, 1, 700, 2, 64, scale=4.0)
    v = normal(rng, dev, dt, 1, 700, 2, 64)
    v *= torch.from_numpy(2.0 ** (np.arange(700) / 64.0)).to(dev).to(dt)[None, :, None, None]
    compare(op, q, k, v, None, None, "f16", dev, None, None, 0, what="growing")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_large_and_equal_scores(dtype, dev):
    # Scores of +-500 (a probability that underflows counts as nothing), and equal ones (each probability 1 / n).
    from afhip import window

    dt, rng = torch_dtype(dtype), np.random.default_rng(7)
    op = window.WindowAttention(2, 1, 64, dtype=dtype)
    q, k, v = normal(rng, dev, dt, 1, 90, 2, 64, scale=22.0), normal(rng, dev, dt, 1, 90, 1, 64, scale=8.0), \
        normal(rng, dev, dt, 1, 90, 1, 64, scale=30.0)
    compare(op, q, k, v, None, None, dtype, dev, None, 0, 0, backward=False, what="large")
    wide = window.WindowAttention(2, 1, 64, right=None, dtype=dtype)
    q.zero_()
    k2, v2 = normal(rng, dev, dt, 1, 3000, 1, 64), normal(rng, dev, dt, 1, 3000, 1, 64)
    compare(wide, q, k2, v2, None, None, dtype, dev, None, None, 0, what="equal")


def test_f16_gradients_keep_their_range(dev):
    # Gradients of 2^-14 and 2^12 times ordinary ones: ds leaves f16's range both ways, the results need not.
    import torch

    from afhip import window

    rng, dt = np.random.default_rng(8), torch.float16
    op = window.WindowAttention(2, 2, 64, dtype="f16")
    q, k = normal(rng, dev, dt, 1, 200, 2, 64), normal(rng, dev, dt, 1, 200, 2, 64)
    for dout_scale, v_scale in ((2.0 ** -9, 2.0 ** -3), (2.0 ** 7, 2.0 ** 6)):
        v = normal(rng, dev, dt, 1, 200, 2, 64, scale=v_scale)
        dout = normal(rng, dev, dt, 1, 200, 2, 64, scale=dout_scale)
        out, lse = op(q, k, v, return_lse=True)
        grads = op.backward(q, k, v, out, lse, dout)
        s = Sequence(f64(q[0]), f64(k[0]), f64(v[0]), 200, 200, None, 0, 0, op.scale, "f16", dout=f64(dout[0]))
        for name, x in zip(("dq", "dk", "dv"), grads):
            holds(x[0], getattr(s, name), getattr(s, name + "_tol"), (name, dout_scale))


def test_backward_against_differences(dev):
    # d loss / dx along a direction, loss = sum out * dout, from the formulas in 64 bits.
    from afhip import window

    rng = np.random.default_rng(9)
    dt = torch_dtype("f32")
    op = window.WindowAttention(4, 2, 32, left=9, right=2, sinks=2, dtype="f32")
    q, k, v = (normal(rng, dev, dt, 1, 50, h, 32) for h in (4, 2, 2))
    dout = normal(rng, dev, dt, 1, 50, 4, 32)
    out, lse = op(q, k, v, return_lse=True)
    grads = op.backward(q, k, v, out, lse, dout)
    args = [f64(x[0]) for x in (q, k, v)]
    loss = lambda *x: (Sequence(*x, 50, 50, 9, 2, 2, op.scale, "f32").out * f64(dout[0])).sum()  # noqa: E731
    for n in range(3):
        direction, step = rng.normal(0, 1, args[n].shape), 1e-5
        ahead, behind = ([a + s * direction if i == n else a for i, a in enumerate(args)] for s in (step, -step))
        difference = (loss(*ahead) - loss(*behind)) / (2 * step)
        terms = f64(grads[n][0]) * direction
        # The third derivative's share, step^2 of values of order 100, and f32's rounding of the terms.
        assert abs(difference - terms.sum()) <= 1e-10 * 1e4 + 1000 * U * np.abs(terms).sum(), n


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_views(dtype, dev):
    # Parts of a projection's rows, heads outside tokens, one entry for all, a given out: the same bits.
    import torch

    from afhip import window

    dt, rng = torch_dtype(dtype), np.random.default_rng(10)
    op = window.WindowAttention(4, 2, 40, left=25, dtype=dtype)
    qkv = normal(rng, dev, dt, 2, 60, 8 * 40)
    q, k, v = (x.unflatten(-1, (-1, 40)) for x in qkv.split([160, 80, 80], -1))
    dout = normal(rng, dev, dt, 2, 60, 4, 40)
    out, lse = op(q.contiguous(), k.contiguous(), v.contiguous(), return_lse=True)
    grads = op.backward(q.contiguous(), k.contiguous(), v.contiguous(), out, lse, dout)
    got, got_lse = op(q, k, v, return_lse=True)
    assert torch.equal(got, out) and torch.equal(got_lse, lse)
    swap = lambda x: x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)  # noqa: E731
    into = torch.empty(2, 4, 60, 40, dtype=dt, device=dev).permute(0, 2, 1, 3)
    assert op(swap(q), swap(k), swap(v), out=into) is into and torch.equal(into, out)
    for a, b in zip(op.backward(q, swap(k), v, into, lse, swap(dout)), grads):
        assert torch.equal(a, b)
    one = [x[:1, :, :1].expand(2, 60, 2, 40) for x in (k, v)]
    want = op(q, *(x.contiguous() for x in one), return_lse=True)
    got = op(q, *one, return_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    dense = op.backward(q, *(x.contiguous() for x in one), *want, dout)
    for a, b in zip(op.backward(q, *one, *got, dout), dense):
        assert torch.equal(a, b)
    broad = dout[:1, :, :1].expand(2, 60, 4, 40)
    for a, b in zip(op.backward(q, k, v, out, lse, broad), op.backward(q, k, v, out, lse, broad.contiguous())):
        assert torch.equal(a, b)


def test_offsets_past_32_bits(dev):
    # Tokens 16 MiB apart: the last keys lie more than 4 GiB from the first.
    import torch

    from afhip import window

    rng, apart = np.random.default_rng(11), 1 << 23
    store = torch.empty(300 * apart, dtype=torch.float16, device=dev)
    far = [store[64 * n:].as_strided((1, 300, 1, 64), (apart, apart, 64, 1)) for n in range(2)]
    near = [normal(rng, dev, torch.float16, 1, 300, 1, 64) for _ in range(2)]
    for x, y in zip(far, near):
        x.copy_(y)
    for tq in (1, 150):
        op = window.WindowAttention(2, 1, 64, dtype="f16")
        q = normal(rng, dev, torch.float16, 1, tq, 2, 64)
        out, lse = op(q, *near, return_lse=True)
        got, got_lse = op(q, *far, return_lse=True)
        assert torch.equal(got, out) and torch.equal(got_lse, lse)
        dout = normal(rng, dev, torch.float16, 1, tq, 2, 64)
        for a, b in zip(op.backward(q, *far, out, lse, dout), op.backward(q, *near, out, lse, dout)):
            assert torch.equal(a, b)


def test_streams_and_graphs(dev):
    # A split call and the way back on another stream, and two graphs of one operator replayed between eager calls.
    import torch

    from afhip import window

    rng, dt = np.random.default_rng(12), torch.float16
    op = window.WindowAttention(8, 2, 128, dtype="f16")
    make = lambda: [normal(rng, dev, dt, 1, n, h, 128) for n, h in ((1, 8), (6000, 2), (6000, 2))]  # noqa: E731
    a, b = make(), make()
    lengths = ints([5500], dev)
    pq, pk, pv, pd = (normal(rng, dev, dt, 1, 100, h, 128) for h in (8, 2, 2, 8))

    def both(x):
        out, lse = op(pq, pk, pv, return_lse=True)
        return [op(*x, key_lengths=lengths), out, lse, *op.backward(pq, pk, pv, out, lse, pd)]

    want = both(a)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = both(a)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graphs, held = [], []
    for x in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(both(x))
        graphs.append(graph)
    for n in range(3):
        for x in (*a, *b, pq, pd):
            x.copy_(normal(rng, dev, dt, *x.shape))
        lengths.fill_(5999 - 1000 * n)
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for x, y in zip((a, b), held):
            assert all(torch.equal(s, t) for s, t in zip(y, both(x))), n


def test_rotary_into_a_cache_then_attention(dev):
    # A layer as it is run: prompts of different lengths into a cache, then steps; every step's output is what
    # attention over the whole sequence gives for its last token.
    import torch

    from afhip import rotary, window

    rng, dt = np.random.default_rng(13), torch.float16
    b, t, h, hk, d, capacity = 2, 70, 8, 2, 64, 90
    turn = rotary.HeadRotary(h, hk, d, norm="rms", dtype="f16")
    turn.prepare(query_scale=np.ones(d, np.float32), key_scale=np.ones(d, np.float32))
    attend = window.WindowAttention(h, hk, d, left=24, right=0, sinks=2, dtype="f16")
    kc = torch.full((b, capacity, hk, d), math.nan, dtype=dt, device=dev)
    vc = kc.clone()
    whole = [normal(rng, dev, dt, b, capacity, n, d) for n in (h, hk, hk)]
    lengths = [70, 51]
    n = ints(lengths, dev)
    q, k, v = turn(*(x[:, :t] for x in whole), lengths=n, k_cache=kc, v_cache=vc)
    outs = [attend(q, k, v, query_lengths=n, key_lengths=n)]
    steps = 15
    for _ in range(steps):
        row = n.long()[:, None, None, None]
        token = [x.gather(1, row.expand(-1, 1, *x.shape[2:])) for x in whole]
        q, k, v = turn(*token, past=n, k_cache=kc, v_cache=vc)
        n = n + 1
        outs.append(attend(q, k, v, key_lengths=n))
    # All at once, each sequence by itself.
    for i in range(b):
        total = lengths[i] + steps
        q, k = turn(whole[0][i:i + 1, :total], whole[1][i:i + 1, :total])
        out, lse = attend(q, k, whole[2][i:i + 1, :total], return_lse=True)
        s = Sequence(f64(q[0]), f64(k[0]), f64(whole[2][i, :total]), total, total, 24, 0, 2, attend.scale, "f16")
        holds(out[0], s.out, s.out_tol, "whole")
        holds(outs[0][i, :lengths[i]], s.out[:lengths[i]], s.out_tol[:lengths[i]], "prompt")
        assert not outs[0][i, lengths[i]:].any()
        for m in range(steps):
            holds(outs[1 + m][i, 0], s.out[lengths[i] + m], s.out_tol[lengths[i] + m], ("step", m))
        assert torch.equal(kc[i, :total], k[0]) and torch.equal(vc[i, :total], whole[2][i, :total])
    # The way back through both, against the chain of their formulas: the gradients agree with those of one call.
    q, k = turn(whole[0][:, :t], whole[1][:, :t])
    out, lse = attend(q, k, whole[2][:, :t], return_lse=True)
    dq, dk, dv = attend.backward(q, k, whole[2][:, :t], out, lse, torch.ones_like(out))
    grads = turn.backward(whole[0][:, :t], whole[1][:, :t], dq, dk)
    assert all(torch.isfinite(x).all() for x in (*grads.values(), dv))


def test_refusals(dev):
    import torch

    from afhip import _lib, window

    rng, dt = np.random.default_rng(14), torch.float16
    op = window.WindowAttention(4, 2, 32, left=5, dtype="f16")
    q, k, v = (normal(rng, dev, dt, 2, n, h, 32) for n, h in ((5, 4), (9, 2), (9, 2)))
    out, lse = op(q, k, v, return_lse=True)

    def refused(match, *args, **kwargs):
        with pytest.raises(_lib.RangeError, match=match):
            op(*args, **kwargs)

    refused("k is on", q, k.cpu(), v)
    refused("torch.float32", q, k.float(), v)
    refused("q has shape", q[0], k, v)
    refused("k has shape", q, k[:1], v)
    refused("v has shape", q, k, v[:, :8])
    refused("contiguous channels", q, k.transpose(2, 3).contiguous().transpose(2, 3), v)
    refused("16 bytes", torch.empty(2, 5, 4, 36, dtype=dt, device=dev)[..., :32], k, v)
    refused("not aligned", torch.empty(2 * 5 * 128 + 8, dtype=dt, device=dev)[4:-4].view(2, 5, 4, 32), k, v)
    refused("repeats one token", q, k[:, :1].expand(2, 9, 2, 32), v)
    refused("query_lengths must be", q, k, v, query_lengths=torch.ones(2, dtype=torch.int64, device=dev))
    refused("key_lengths must be", q, k, v, key_lengths=ints([1, 2, 3], dev))
    refused("key_lengths is on", q, k, v, key_lengths=torch.ones(2, dtype=torch.int32))
    refused("out has shape", q, k, v, out=k)
    refused("repeats one entry", q, k, v, out=q[:1].expand(2, 5, 4, 32))
    refused("positive", q[:, :0], k, v)
    refused("positive", q, k[:, :0], v[:, :0])
    for args in ((q, k, v, out, lse[:1], q), (q, k, v, out, lse.half(), q), (q, k, v, out, lse, k),
                 (q, k, v, k, lse, q), (q, k, v, out, lse.cpu(), q)):
        with pytest.raises(_lib.RangeError):
            op.backward(*args)
    for bad in (dict(dtype="bf16"), dict(left=-3), dict(sinks=-1), dict(scale=0.0), dict(scale=math.nan)):
        with pytest.raises(_lib.RangeError):
            window.WindowAttention(4, 2, 32, **bad)
    for heads in ((4, 3, 32), (4, 2, 33), (4, 2, 136), (4, 2, 0), (0, 1, 32)):
        with pytest.raises(_lib.RangeError):
            window.WindowAttention(*heads)
    many = torch.zeros(1, 1, 1, 8, dtype=dt, device=dev).expand(1 << 24, 1, 1, 8)
    with pytest.raises(_lib.RangeError, match="too many for one launch"):
        window.WindowAttention(1, 1, 8, dtype="f16")(many, many, many)
