"""HeadRotary on the GPU against its formulas in 64 bits.

Tolerances. U = 2^-24 is half a step of f32 relative to the value, T half a
step of the tensors' type. With S the largest |x| r |w| + |c| of a head's row
(r the reciprocal root, 1 without a norm), the forward pass errs at most
  4.5 U r from the sum of squares (8 additions and a product, halved by the
  root), 2 U from root and reciprocal, 9 U from the mean and its subtraction,
  3 U from the products and the sum, 4 U from a cosine or sine (2 steps of
  the function, and an argument of up to pi that is off by 2^-25 pi),
  3 U from the rotation's products and sum,
of S for each of two terms: 2 * 25.5 U S < 64 U S, times the rotation's
factor, and T |y| (f16: plus 2^-25 where it is subnormal) from the last
rounding. The way back has the same terms on G = r max |g w| (its mean
products: two more reductions, 9 U each), with xhat of at most sqrt(D):
96 U G (1 + sqrt(D)) + T |dx|. The vectors' gradients are sums of n terms in
f32 partial sums of at most 8 + 6 + 2 additions (a workgroup's rows of a
lane), then in 64 bits: (rows of a lane + 32) U sum |terms|.
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


def turn(x, angles, scale, layout, r, sign=1):
    """x [..., D] by angles [..., r / 2], f64."""
    y = x.copy()
    a = slice(0, r // 2) if layout == "half" else slice(0, r, 2)
    b = slice(r // 2, r) if layout == "half" else slice(1, r, 2)
    c, s = np.cos(angles) * scale, np.sin(angles) * scale * sign
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def reference(x, positions, freq, scale, layout, norm, w, c, eps):
    """(y, size): the rows in 64 bits, and S for each of them."""
    r = np.ones(x.shape[:-1] + (1,))
    n = x
    if norm is not None:
        n = x - (x.mean(-1, keepdims=True) if norm == "layer" else 0.0)
        r = 1 / np.sqrt((n * n).mean(-1, keepdims=True) + eps)
        n = n * r * w
    size = (np.abs(x) * r * (1 if w is None else np.abs(w)) + (0 if c is None else np.abs(c))).max(-1, keepdims=True)
    if c is not None:
        n = n + c
    return turn(n, positions[:, :, None, None] * freq, scale, layout, 2 * len(freq)), size * max(1.0, abs(scale))


def backward_reference(x, g, positions, freq, scale, layout, norm, w, eps):
    """(dx, dw, dc, G, sum |terms of dw|, sum |terms of dc|)."""
    g = turn(g, positions[:, :, None, None] * freq, scale, layout, 2 * len(freq), -1)
    if norm is None:
        return g, None, None, np.abs(g).max(-1, keepdims=True) + 0 * x[..., :1], None, None
    n = x - (x.mean(-1, keepdims=True) if norm == "layer" else 0.0)
    r = 1 / np.sqrt((n * n).mean(-1, keepdims=True) + eps)
    n = n * r
    gw = g * w
    dx = gw - n * (gw * n).mean(-1, keepdims=True)
    if norm == "layer":
        dx = dx - gw.mean(-1, keepdims=True)
    size = (np.abs(gw).max(-1, keepdims=True)) * r
    return (r * dx, (g * n).sum((0, 1, 2)), g.sum((0, 1, 2)), size, np.abs(g * n).sum((0, 1, 2)),
            np.abs(g).sum((0, 1, 2)))


# batch, tokens, query heads, key heads, head_dim, rotary_dim, layout, norm, dtype
CASES = [
    (1, 1, 1, 1, 8, 8, "half", "rms", "f32"),
    (2, 3, 4, 2, 16, 8, "interleaved", "layer", "f32"),
    (2, 33, 8, 8, 32, 16, "half", "layer", "f32"),
    (1, 130, 6, 3, 40, 40, "half", "rms", "f16"),
    (3, 17, 4, 1, 64, 64, "interleaved", "rms", "f16"),
    (2, 29, 5, 7, 80, 24, "half", None, "f32"),
    (1, 700, 32, 8, 128, 128, "half", "rms", "f16"),
    (2, 1500, 3, 1, 128, 64, "interleaved", "layer", "f16"),
    (1, 4, 2, 2, 64, 0, "half", "rms", "f32"),
    (70, 1, 16, 2, 24, 24, "interleaved", None, "f16"),
    # Odd multiples of 4: the last pairs share a lane with channels that do not turn.
    (2, 37, 6, 3, 40, 20, "half", "rms", "f16"),
    (1, 45, 8, 2, 40, 20, "interleaved", "layer", "f32"),
    (2, 19, 3, 1, 8, 4, "half", "layer", "f32"),
    (1, 90, 4, 2, 128, 100, "half", "layer", "f16"),
    (3, 11, 2, 2, 128, 124, "interleaved", "rms", "f32"),
    (2, 21, 4, 4, 80, 76, "half", None, "f32"),
]


def build(case, seed, dev, **kwargs):
    import torch

    from afhip import rotary

    b, t, h, hk, d, r, layout, norm, dtype = case
    rng = np.random.default_rng(seed)
    freq = 10000.0 ** (-np.arange(0, r, 2) / max(r, 1))
    scale = kwargs.pop("rotation_scale", 1.25)
    op = rotary.HeadRotary(h, hk, d, rotary_dim=r, layout=layout, norm=norm, dtype=dtype, frequencies=freq,
                           rotation_scale=scale, **kwargs)
    vectors = {}
    if norm is not None:
        vectors = {"query_scale": rng.normal(1, 0.2, d), "key_scale": rng.normal(1, 0.2, d)}
        if norm == "layer":
            vectors |= {"query_offset": rng.normal(0, 0.2, d), "key_offset": rng.normal(0, 0.2, d)}
        vectors = {n: v.astype(np.float32) for n, v in vectors.items()}
        op.prepare(**vectors)
    dt = torch.float16 if dtype == "f16" else torch.float32
    make = lambda *shape: torch.from_numpy(rng.normal(0, 1, shape).astype(np.float32)).to(dev).to(dt)  # noqa: E731
    q, k, v = make(b, t, h, d), make(b, t, hk, d), make(b, t, hk, d)
    return op, q, k, v, freq, scale, vectors, rng, make


def f64(x):
    return x.double().cpu().numpy()


def ints(values, dev):
    import torch

    return torch.tensor(values, dtype=torch.int32, device=dev)


def expected(x, positions, freq, scale, case, vectors, side, eps=1e-5):
    _, _, _, _, d, r, layout, norm, dtype = case
    w, c = vectors.get(side + "_scale"), vectors.get(side + "_offset")
    y, size = reference(f64(x), positions, freq, scale, layout, norm, None if w is None else w.astype(np.float64),
                        None if c is None else c.astype(np.float64), eps)
    return y, 64 * U * size + T[dtype] * np.abs(y) + SMALL[dtype]


def holds(got, want, tolerance, what):
    off = np.abs(f64(got) - want)
    assert np.isfinite(off).all(), what
    assert (off <= tolerance).all(), (what, float((off / tolerance).max()))


@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward(case, dev):
    b, t = case[:2]
    print("rotary forward", case, flush=True)
    op, q, k, v, freq, scale, vectors, rng, _ = build(case, 1, dev)
    got_q, got_k = op(q, k)
    positions = np.broadcast_to(np.arange(t, dtype=np.float64), (b, t))
    holds(got_q, *expected(q, positions, freq, scale, case, vectors, "query"), "q")
    holds(got_k, *expected(k, positions, freq, scale, case, vectors, "key"), "k")


@pytest.mark.parametrize("case", CASES, ids=str)
def test_cache_lengths_and_past(case, dev):
    # Rows of the cache that are not written keep their bits; tokens past the length give zeros; a token whose row
    # lies past the cache's end (the last sequence's) or before its start is not written.
    import torch

    b, t, h, hk, d, r, layout, norm, dtype = case
    print("rotary cache", case, flush=True)
    op, q, k, v, freq, scale, vectors, rng, make = build(case, 2, dev)
    capacity = t + 9
    lengths = [max(0, t - (i * 5) % (t + 1)) for i in range(b)]
    past = [(i * 4) % 10 for i in range(b)]
    past[-1] = 10 if b > 1 else 9
    if b > 2:
        past[1] = -2
    kc, vc = make(b, capacity, hk, d), make(b, capacity, hk, d)
    k_want, v_want = kc.clone(), vc.clone()
    got_q, got_k, got_v = op(q, k, v, past=ints(past, dev), lengths=ints(lengths, dev), k_cache=kc, v_cache=vc)
    assert got_k is kc and got_v is vc
    positions = np.arange(t, dtype=np.float64)[None] + np.array(past, dtype=np.float64)[:, None]
    want, tolerance = expected(q, positions, freq, scale, case, vectors, "query")
    kw, kt = expected(k, positions, freq, scale, case, vectors, "key")
    written = torch.zeros(b, capacity, dtype=torch.bool)
    for i in range(b):
        want[i, lengths[i]:], tolerance[i, lengths[i]:] = 0, 0
        for j in range(lengths[i]):
            row = past[i] + j
            if 0 <= row < capacity:
                written[i, row] = True
                holds(kc[i, row], kw[i, j], kt[i, j], ("k", i, j))
                v_want[i, row] = v[i, j]
    holds(got_q, want, tolerance, "q")
    assert torch.equal(vc, v_want)
    assert torch.equal(kc[~written.to(dev)], k_want[~written.to(dev)])


def test_lengths_without_a_cache(dev):
    case = (3, 6, 2, 2, 32, 32, "half", "rms", "f16")
    op, q, k, v, freq, scale, vectors, _, _ = build(case, 3, dev)
    lengths = [0, 6, 4]
    q[0], k[0] = math.nan, math.inf  # past the length: not looked at
    got_q, got_k = op(q, k, lengths=ints(lengths, dev))
    for x, got, side in ((q, got_q, "query"), (k, got_k, "key")):
        want, tolerance = expected(x, np.broadcast_to(np.arange(6.0), (3, 6)), freq, scale, case, vectors, side)
        for i, n in enumerate(lengths):
            want[i, n:], tolerance[i, n:] = 0, 0
        holds(got, want, tolerance, side)


def test_far_positions(dev):
    # A product of 32 bits would turn these by 0.06 rad too much or too little.
    import torch

    case = (1, 4, 1, 1, 64, 64, "half", None, "f32")
    op, q, k, v, freq, scale, vectors, _, _ = build(case, 4, dev)
    at = [[1_000_003, 2 ** 31 - 1, 123_456_789, -77_777]]
    got_q, _ = op(q, k, positions=torch.tensor(at, dtype=torch.int32, device=dev))
    # An angle of 2^31 in 64 bits is off by half a step there, 2^-23.
    want, tolerance = expected(q, np.array(at, dtype=np.float64), freq, scale, case, vectors, "query")
    holds(got_q, want, tolerance + 4 * 2.0 ** -22 * np.abs(want).max(), "q")
    got, _ = op(q, k, past=ints([2 ** 31 - 3], dev))
    want, tolerance = expected(q, np.array([[2.0 ** 31 - 3 + i for i in range(4)]]), freq, scale, case, vectors,
                               "query")
    holds(got, want, tolerance + 4 * 2.0 ** -22 * np.abs(want).max(), "past")


def test_views_and_in_place(dev):
    # q, k and v side by side as a projection writes them, heads outside tokens, and in place.
    import torch

    case = (2, 37, 4, 2, 64, 64, "half", "rms", "f16")
    op, q, k, v, freq, scale, vectors, _, make = build(case, 5, dev)
    plain_q, plain_k = op(q, k)
    qkv = torch.cat([x.flatten(2) for x in (q, k, v)], -1)
    views = [x.unflatten(-1, (-1, 64)) for x in qkv.split([256, 128, 128], -1)]
    assert not views[0].is_contiguous()
    got_q, got_k = op(views[0], views[1])
    assert torch.equal(got_q, plain_q) and torch.equal(got_k, plain_k)
    outside = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    into = torch.empty(2, 4, 37, 64, dtype=torch.float16, device=dev).permute(0, 2, 1, 3)
    got_q, _ = op(outside, k, q_out=into)
    assert got_q is into and torch.equal(into, plain_q)
    # In place, in the projection's rows.
    op(views[0], views[1], q_out=views[0], k_out=views[1])
    assert torch.equal(views[0], plain_q) and torch.equal(views[1], plain_k)
    assert torch.equal(views[2], v)
    # A head that stands for all, a batch entry too.
    one = q[:1, :, :1].expand(2, 37, 4, 64)
    got_q, _ = op(one, k)
    again, _ = op(one.contiguous(), k)
    assert torch.equal(got_q, again)


@pytest.mark.parametrize("case", CASES, ids=str)
def test_backward(case, dev):
    import torch

    b, t, h, hk, d, r, layout, norm, dtype = case
    print("rotary backward", case, flush=True)
    op, q, k, v, freq, scale, vectors, _, make = build(case, 6, dev)
    gq, gk = make(b, t, h, d), make(b, t, hk, d)
    lengths = [max(0, t - (i * 7) % (t + 1)) for i in range(b)]
    past = [3 * i for i in range(b)]
    got = op.backward(q, k, gq, gk, past=ints(past, dev), lengths=ints(lengths, dev))
    again = op.backward(q, k, gq, gk, past=ints(past, dev), lengths=ints(lengths, dev))
    assert set(got) == {"dq", "dk"} | {"d" + n for n in vectors}
    assert all(torch.equal(got[n], again[n]) for n in got)
    positions = np.arange(t, dtype=np.float64)[None] + np.array(past, dtype=np.float64)[:, None]
    live = (np.arange(t)[None] < np.array(lengths)[:, None])[:, :, None, None]
    for x, g, side, name in ((q, gq, "query", "dq"), (k, gk, "key", "dk")):
        w = vectors.get(side + "_scale")
        dx, dw, dc, size, sw, sc = backward_reference(f64(x), np.where(live, f64(g), 0), positions, freq, scale,
                                                      layout, norm, None if w is None else w.astype(np.float64), 1e-5)
        tolerance = 96 * U * size * (1 + math.sqrt(d)) * abs(scale) + T[dtype] * np.abs(dx) + SMALL[dtype]
        holds(got[name], np.where(live, dx, 0), np.where(live, tolerance, 0), name)
        # A lane's rows: its workgroup's share, at most all of them.
        rows = b * t * (h if side == "query" else hk)
        per_lane = min(rows, 16 * 16)
        # Each term errs by at most 32 U of |g xhat| (64 U S relative to its parts, halved: one factor).
        if norm is not None:
            holds(got[f"d{side}_scale"], dw, (per_lane + 96) * U * (sw + 1e-30), side + " scale")
        if norm == "layer":
            holds(got[f"d{side}_offset"], dc, (per_lane + 96) * U * (sc + 1e-30), side + " offset")


def test_backward_against_differences(dev):
    # Of the forward pass in 64 bits: d loss / dx along a direction, for loss = sum y g.
    import torch

    case = (1, 5, 2, 1, 32, 16, "interleaved", "layer", "f32")
    op, q, k, v, freq, scale, vectors, rng, make = build(case, 7, dev)
    gq, gk = make(1, 5, 2, 32), make(1, 5, 1, 32)
    got = op.backward(q, k, gq, gk)
    positions = np.arange(5.0)[None]
    w, c = vectors["query_scale"].astype(np.float64), vectors["query_offset"].astype(np.float64)
    loss = lambda x, w, c: (reference(x, positions, freq, scale, "interleaved", "layer", w, c, 1e-5)[0]  # noqa: E731
                            * f64(gq)).sum()
    x, step = f64(q), 1e-6
    for name, args, n in (("dq", (x, w, c), 0), ("dquery_scale", (x, w, c), 1), ("dquery_offset", (x, w, c), 2)):
        direction = rng.normal(0, 1, args[n].shape)
        ahead, behind = ([a + s * direction if i == n else a for i, a in enumerate(args)] for s in (step, -step))
        difference = (loss(*ahead) - loss(*behind)) / (2 * step)
        along = (f64(got[name]) * direction).sum()
        # Second differences: step^2 on values of order 1; f32 gradients: 96 U of the terms' magnitudes.
        assert abs(difference - along) <= 1e-8 * 200 + 200 * U * (np.abs(f64(got[name]) * direction)).sum() + 1e-4, name


def test_sums_of_many_tokens(dev):
    # More tiles than the way back has workgroups; f32 partial sums, then 64 bits.
    case = (2, 9001, 4, 1, 32, 32, "half", "rms", "f16")
    op, q, k, v, freq, scale, vectors, _, make = build(case, 8, dev)
    gq, gk = make(2, 9001, 4, 32), make(2, 9001, 1, 32)
    got = op.backward(q, k, gq, gk)
    positions = np.broadcast_to(np.arange(9001.0), (2, 9001))
    for x, g, side in ((q, gq, "query"), (k, gk, "key")):
        _, dw, _, _, sw, _ = backward_reference(f64(x), f64(g), positions, freq, scale, "half", "rms",
                                                vectors[side + "_scale"].astype(np.float64), 1e-5)
        holds(got[f"d{side}_scale"], dw, (256 + 96) * U * sw, side)


def test_streams_and_graphs(dev):
    # On another stream than the tensors' own; captured with the way back, and replayed on new inputs between eager calls.
    import torch

    case = (2, 40, 4, 2, 64, 64, "half", "rms", "f16")
    op, q, k, v, freq, scale, vectors, _, make = build(case, 9, dev)
    kc, vc = make(2, 64, 2, 64), make(2, 64, 2, 64)
    past = ints([3, 20], dev)
    gq, gk = make(2, 40, 4, 64), make(2, 40, 2, 64)
    side = torch.cuda.Stream()
    want = [x.clone() for x in op(q, k, v, past=past, k_cache=kc, v_cache=vc)]
    back = op.backward(q, k, gq, gk, past=past)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = op(q, k, v, past=past, k_cache=kc, v_cache=vc)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = op(q, k, v, past=past, k_cache=kc, v_cache=vc)
        held_back = op.backward(q, k, gq, gk, past=past)
    for n in range(3):
        q.copy_(make(2, 40, 4, 64))
        k.copy_(make(2, 40, 2, 64))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        got_back = {name: x.clone() for name, x in held_back.items()}
        want = op(q, k, v, past=past, k_cache=kc, v_cache=vc)
        back = op.backward(q, k, gq, gk, past=past)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), n
        assert all(torch.equal(got_back[name], back[name]) for name in back), n


def test_refusals(dev):
    import torch

    from afhip import _lib, rotary

    case = (2, 5, 4, 2, 32, 32, "half", "rms", "f16")
    op, q, k, v, freq, scale, vectors, _, make = build(case, 10, dev)
    kc, vc = make(2, 9, 2, 32), make(2, 9, 2, 32)

    def refused(match, *args, **kwargs):
        with pytest.raises(_lib.RangeError, match=match):
            op(*args, **kwargs)

    refused("q is on", q.cpu(), k)
    refused("torch.float32", q.float(), k)
    refused("q has shape", q[0], k)
    refused("k has shape", q, k[:, :4])
    refused("k has shape", q, q)
    refused("contiguous channels", q.transpose(2, 3).contiguous().transpose(2, 3), k)
    refused("16 bytes", torch.empty(2, 5, 4, 36, dtype=q.dtype, device=dev)[..., :32], k)
    refused("not aligned", torch.empty(2 * 5 * 128 + 8, dtype=q.dtype, device=dev)[4:-4].view(2, 5, 4, 32), k)
    refused("repeats one token", q[:, :1].expand(2, 5, 4, 32), k)
    refused("past must be", q, k, past=torch.zeros(2, dtype=torch.int64, device=dev))
    refused("past is on", q, k, past=torch.zeros(2, dtype=torch.int32))
    refused("lengths must be", q, k, lengths=ints([1], dev))
    refused("positions must be", q, k, positions=ints([1, 2], dev))
    refused("v is taken", q, k, v)
    refused("v and v_cache", q, k, v, k_cache=kc)
    refused("v and v_cache", q, k, k_cache=kc, v_cache=vc)
    refused("k_out is not taken", q, k, v, k_cache=kc, v_cache=vc, k_out=k)
    refused("k_cache has shape", q, k, v, k_cache=kc[:1], v_cache=vc)
    refused("holds no tokens", q, k, v, k_cache=kc[:, :0], v_cache=vc[:, :0])
    refused("repeats one entry", q, k, q_out=q[:1].expand(2, 5, 4, 32))
    refused("positive", q[:, :0], k[:, :0])
    with pytest.raises(_lib.RangeError, match="dq_out has shape"):
        op.backward(q, k, q[:1], k)
    fresh = rotary.HeadRotary(4, 2, 32, norm="rms", dtype="f16")
    with pytest.raises(_lib.RangeError, match="prepare"):
        fresh(q, k)
    for bad in (dict(), dict(query_scale=np.ones(32, np.float32)),
                dict(query_scale=np.ones(31, np.float32), key_scale=np.ones(32, np.float32)),
                dict(query_scale=np.ones(32, np.float32), key_scale=np.ones(32, np.float32),
                     key_offset=np.ones(32, np.float32))):
        with pytest.raises(_lib.RangeError):
            fresh.prepare(**bad)
    for bad in (dict(dtype="bf16"), dict(layout="other"), dict(norm="batch"), dict(rotary_dim=10),
                dict(frequencies=np.ones(3))):
        with pytest.raises(_lib.RangeError):
            rotary.HeadRotary(4, 2, 32, **{"dtype": "f16", **bad})
    many = torch.zeros(1, 1, 1, 8, dtype=q.dtype, device=dev).expand(1 << 23, 1, 1, 8)
    with pytest.raises(_lib.RangeError, match="too many for one launch"):
        rotary.HeadRotary(1, 1, 8, dtype="f16")(many, many)
