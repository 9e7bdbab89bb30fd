"""The correlation losses on the MI355X (cross entropy and distillation,
forward and backward) against the float64 oracle.

Tolerances, with u = 2^-24, h = half a step of the features' type.
Logits: a product of two features is exact in fp32, D of them are added in
fp32: |error| <= D u sum_d |x_d y_d| scale / T =: r (its largest over the
row's keys).  lse: r, plus Q u for at most Q fp32 additions of the sum, plus a
few roundings of the value.  loss: the two logit errors, T^2 times.
Weights: p off by a factor of at most 1 + r + Q u + 8 u (1 + |lse|); p - pi
and its product with g a rounding each, then one rounding to the features'
type: h |ds| (fp16 weights are scaled to 2^13 times the edge's largest |g|
share, so what underflows is below 2^-38 of it).  Gradients: these sums over
the other rows, n fp32 additions of them, one rounding at the end.
An edge and its reverse with upstream gradients >= 0 share one exponential:
the weights are products of three powers of two whose exponents are below
60 + |log2 g| + 1.5 |lse| each and are rounded once: PAIR u more, relative to p,
and what underflows is below 2^-86 of a probability."""
import numpy as np
import pytest
import torch

from gpu_util import host
from oracle import corr_loss as oc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
PAIR = 256
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _problem(seed, dt, K, E, N1, P, N2, Q, D, amp=1.0, shared=False, gscale=1.0):
    """Random frames; targets anywhere, some rows without one."""
    rng = np.random.default_rng(seed)
    f = lambda n, r: torch.from_numpy(rng.normal(size=(n, r, D)) * amp).to(dt).to(DEV)
    a = f(N1, P)
    b = a if shared else f(N2, Q)
    f1 = rng.integers(0, N1, E).astype(np.int32)
    f2 = rng.integers(0, N1 if shared else N2, E).astype(np.int32)
    idx = rng.random((E, P, Q)).argsort(-1)[..., :max(1, K)].astype(np.int32)
    idx[rng.random((E, P)) < 0.2] = -1
    idx[rng.random(idx.shape) < 0.1] = -1
    logits = (3 * rng.normal(size=idx.shape)).astype(np.float32) if K else None
    g = (rng.normal(size=(E, P)) * gscale).astype(np.float32)
    return a, b, f1, f2, idx, logits, g


def _t(x):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


def _run(a, b, f1, f2, idx, logits, g, shared, scale, T):
    from droid_mi355x import corr_cross_entropy, corr_distillation
    leaves = [t.detach().clone().requires_grad_() for t in ([a] if shared else [a, b])]
    k = (leaves[0], None if shared else leaves[1], _t(f1), _t(f2))
    loss = (corr_cross_entropy(*k, _t(idx[..., 0]), scale) if logits is None
            else corr_distillation(*k, _t(idx), _t(logits), scale, T))
    return loss.detach(), torch.autograd.grad(loss, leaves, _t(g))


def _check(dt, a, b, f1, f2, idx, logits, g, shared, scale, T, loss, grads, more=0):
    A, B = host(a.double()), host(b.double())
    T = T if logits is not None else 1.0
    D, Q, h = A.shape[-1], B.shape[1], torch.finfo(dt).eps / 2
    want, d1, d2, per_edge = oc.corr_loss(A, B, f1, f2, idx, logits, scale, T, g)
    e1, e2 = np.zeros_like(d1), np.zeros_like(d2)
    for e, (ds, p, q, lse) in enumerate(per_edge):
        x, y = np.abs(A[f1[e]]), np.abs(B[f2[e]])
        r = D * U * (x @ y.T).max(1) * scale / T
        tol = T * T * (2 * r + U * (Q + 8 + 8 * np.abs(lse) + 2 * (x @ y.T).max(1) * scale / T)) + 1e-6 * T * T * (
            logits is not None)                       # logf / expf of the teacher's weights: K entries, a few u each
        assert (np.abs(host(loss)[e] - want[e]) <= tol).all(), e
        ge = np.abs(g[e])[:, None] * T * scale
        rel = (r + Q * U + 8 * U * (1 + np.abs(lse)) + more * U)[:, None]
        # rows with a target: also where p - pi is exactly 0 (one key: p = 1 up to its error), left-out rows are exact
        on = (q.max(1, keepdims=True) > 0)
        floor = np.abs(g).max() * T * scale * 2.0 ** -38 if dt == torch.float16 else 0.0
        err = np.where(on, h * np.abs(ds) + ge * (p * rel + 4 * U * (p + q)) + floor, 0.0)
        mag = np.abs(ds) + err
        e1[f1[e]] += (err + (Q + 8) * U * mag) @ y
        e2[f2[e]] += (err + (x.shape[0] + 8) * U * mag).T @ x
    if shared:
        d1, e1 = d1 + d2, e1 + e2
    sub = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -126
    for got, d, e in zip(grads, (d1, d2), (e1, e2)):
        assert got.dtype == dt
        assert (np.abs(host(got.double()) - d) <= 1.01 * e + (h + 4 * U) * np.abs(d) + sub).all()


SIZES = [  # E, N1, P, N2, Q, D
    (1, 1, 1, 1, 1, 8), (2, 1, 1, 2, 65, 32), (3, 2, 130, 2, 63, 64), (2, 2, 64, 1, 128, 128), (4, 3, 257, 2, 200, 128),
    (2, 2, 33, 2, 500, 72), (1, 1, 129, 1, 1, 256), (3, 2, 140, 3, 129, 200), (300, 4, 3, 5, 70, 16)]


@pytest.mark.parametrize("K", [0, 1, 4, 7, 16, 64])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("E,N1,P,N2,Q,D", SIZES)
def test_separate_features(E, N1, P, N2, Q, D, dtype, K):
    if K > Q:
        pytest.skip("more targets than keys")
    dt, T = TYPES[dtype], 1.0 if K < 7 else 2.0
    p = _problem(E * P + Q + K, dt, K, E, N1, P, N2, Q, D)
    loss, grads = _run(*p, False, 1 / 16, T)
    _check(dt, *p, False, 1 / 16, T, loss, grads)


@pytest.mark.parametrize("K", [0, 5])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("E,N,P,D", [(6, 3, 190, 128), (12, 4, 70, 64), (3, 1, 300, 128), (2, 2, 1, 8)])
def test_shared_features(E, N, P, D, dtype, K):
    """A frame graph: the same features are queries and keys (self edges among them)."""
    if K > P:
        pytest.skip("more targets than keys")
    dt = TYPES[dtype]
    p = _problem(E + P, dt, K, E, N, P, N, P, D, shared=True)
    loss, grads = _run(*p, True, 1 / 16, 1.0)
    _check(dt, *p, True, 1 / 16, 1.0, loss, grads)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("gscale", [1e-7, 1.0, 1e4])
def test_peaked_softmax_keeps_the_small_difference(dtype, gscale):
    """Well-trained features: p near 1 at the target, the gradient is the small
    p - 1; upstream gradients of a mean and of a large loss scale."""
    dt = TYPES[dtype]
    a, b, f1, f2, idx, _, g = _problem(5, dt, 0, 2, 2, 100, 2, 150, 128, shared=False, gscale=gscale)
    b = b.clone()
    for e in range(2):
        for r in range(100):
            if idx[e, r, 0] >= 0 and f1[e] == 0:
                idx[e, r, 0] = r
    b[:, :100] = a[:1]
    p = (a, b, f1, f2, idx, None, g)
    loss, grads = _run(*p, False, 1 / 16, 1.0)
    out = torch.finfo(dt).max
    if all(t.abs().max() < out for t in grads):
        _check(dt, *p, False, 1 / 16, 1.0, loss, grads)


def test_rows_without_targets():
    """NaN and infinities in the features of left-out rows, edges without any
    target onto a frame of NaN, empty places and -inf / lowest logits."""
    dt = torch.float16
    a, b, f1, f2, idx, logits, g = _problem(7, dt, 3, 4, 2, 150, 3, 90, 64)
    f1[:], f2[:] = [0, 1, 0, 1], [0, 1, 1, 2]
    idx[3] = -1                                   # the only edge onto frame 2 of b
    idx[0, 10:20], idx[2, 10:20] = -1, -1         # frame 0 of a: rows without a target in both of its edges
    logits[1, 0], logits[1, 1, 0] = -np.inf, -np.inf
    logits[1, 2] = np.finfo(np.float32).min
    clean_a, clean_b = a.clone(), b.clone()
    clean_a[0, 10:20], clean_b[2] = 0.0, 0.0
    a, b = a.clone(), b.clone()
    a[0, 10:20], b[2] = float("nan"), float("nan")
    a[0, 13], b[2, 5] = float("inf"), float("-inf")
    for xent in (False, True):
        i, l = (idx[..., :1], None) if xent else (idx, logits)
        loss, grads = _run(a, b, f1, f2, i, l, g, False, 1 / 16, 1.0)
        _check(dt, clean_a, clean_b, f1, f2, i, l, g, False, 1 / 16, 1.0, loss, grads)
        assert not grads[0][0, 10:20].any() and not grads[1][2].any() and not loss[3].any()
    # nothing at all to learn
    loss, grads = _run(a, b, f1, f2, np.full_like(idx, -1), logits, g, False, 1 / 16, 1.0)
    assert not loss.any() and not grads[0].any() and not grads[1].any()


def test_wrong_targets_and_edges_answer_nan():
    dt = torch.bfloat16
    a, b, f1, f2, idx, _, g = _problem(8, dt, 0, 3, 2, 40, 2, 50, 64)
    idx[:] = 5
    idx[0, 3, 0] = 50
    good = f2.copy()
    f2[1], f1[2] = 2, -1
    loss, grads = _run(a, b, f1, f2, idx, None, g, False, 1 / 16, 1.0)
    bad = torch.zeros((3, 40), dtype=torch.bool)
    bad[0, 3], bad[1], bad[2] = True, True, True
    assert torch.equal(loss.isnan().cpu(), bad)
    assert grads[0][f1[0], 3].isnan().all() and grads[1][good[0]].isnan().any()
    other = [n for n in range(2) if n != f1[0]]
    assert not grads[0][other].isnan().any()


def test_equal_bits_streams_and_graph_replay():
    """Repeatable bit for bit; on a side stream; captured, replayed on new
    inputs with eager work between."""
    import droid_backends as nb
    ps = [_problem(s, torch.float16, 4, 5, 3, 140, 3, 140, 128, shared=True) for s in range(3)]
    f1, f2 = _t(ps[0][2]), _t(ps[0][3])

    def both(x, i, l, g):
        loss, lse, prob = nb.corr_loss_forward(x, None, f1, f2, i, l)
        return loss, nb.corr_loss_backward(g, x, None, f1, f2, i, lse, prob)[0]

    ins = [(p[0], _t(p[4]), _t(p[5]), _t(p[6])) for p in ps]
    want = [both(*i) for i in ins]
    buf = [t.clone() for t in ins[0]]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both(*buf)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(got, want[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(*buf)
    for k in (1, 2, 0, 1):
        for dst, src in zip(buf, ins[k]):
            dst.copy_(src)
        graph.replay()
        both(*ins[2])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want[k])), k


def test_wanted_gradients_broadcast_upstream_and_map_shapes():
    """Only the gradients that are asked for; an expanded upstream gradient;
    (frames, H, W, D) maps with (edges, H, W) targets."""
    from droid_mi355x import corr_cross_entropy
    a, b, f1, f2, idx, _, g = _problem(11, torch.bfloat16, 0, 3, 2, 60, 2, 77, 64)
    a4, b4 = a.view(2, 6, 10, 64), b.view(2, 7, 11, 64)
    t = _t(idx[..., 0]).view(3, 6, 10)
    ref = _run(a, b, f1, f2, idx, None, np.ones_like(g), False, 1 / 16, 1.0)[1]
    x, y = a4.clone().requires_grad_(), b4.clone().requires_grad_()
    gx, gy = torch.autograd.grad(corr_cross_entropy(x, y, _t(f1), _t(f2), t).sum(), [x, y])
    assert torch.equal(gx.view_as(ref[0]), ref[0]) and torch.equal(gy.view_as(ref[1]), ref[1])
    for keep in (0, 1):
        x, y = a4.clone(), b4.clone()
        leaf = (x, y)[keep].requires_grad_()
        got, = torch.autograd.grad(corr_cross_entropy(x, y, _t(f1), _t(f2), t).sum(), [leaf])
        # a share of the other split of the streamed rows: the same sums in another order
        np.testing.assert_allclose(host(got.float()), host((gx, gy)[keep].float()), rtol=2.0 ** -7, atol=1e-5)
    with torch.no_grad():
        assert corr_cross_entropy(a4, b4, _t(f1), _t(f2), t).shape == (3, 6, 10)


def test_device_refusals_and_empty_calls():
    import droid_backends as nb
    a, b, f1, f2, idx, logits, g = _problem(2, torch.float16, 3, 2, 2, 20, 2, 30, 16)
    ok = dict(fmap1=a, fmap2=b, f1=_t(f1), f2=_t(f2), idx=_t(idx), logits=_t(logits))
    bad = [dict(fmap1=a.float()), dict(fmap2=b.bfloat16()), dict(f1=_t(f1).long()), dict(f2=_t(f2)[:1]),
           dict(idx=_t(idx).long()), dict(idx=_t(idx)[:, :10].contiguous()), dict(logits=_t(logits).half()),
           dict(logits=_t(logits)[..., :2].contiguous()), dict(fmap1=a[..., :12].contiguous()),
           dict(fmap2=b.transpose(0, 1)), dict(f1=_t(f1).cpu()), dict(scale=0.0), dict(temperature=-1.0),
           dict(fmap1=a[0]), dict(idx=_t(idx)[..., :0].contiguous(), logits=_t(logits)[..., :0].contiguous())]
    for kw in bad:
        with pytest.raises((RuntimeError, TypeError)):
            nb.corr_loss_forward(**{**ok, **kw})
    loss, lse, prob = nb.corr_loss_forward(**ok)
    with pytest.raises(RuntimeError):
        nb.corr_loss_backward(_t(g).half(), a, b, _t(f1), _t(f2), _t(idx), lse, prob)
    with pytest.raises(RuntimeError):
        nb.corr_loss_backward(_t(g)[:, :3].contiguous(), a, b, _t(f1), _t(f2), _t(idx), lse, prob)
    e = torch.empty(0, dtype=torch.int32, device=DEV)
    loss, lse, prob = nb.corr_loss_forward(a, b, e, e, torch.empty((0, 20), dtype=torch.int32, device=DEV))
    assert loss.shape == (0, 20) and prob is None
    d1, d2 = nb.corr_loss_backward(loss, a, b, e, e, torch.empty((0, 20), dtype=torch.int32, device=DEV), lse)
    assert d1.shape == a.shape and d2.shape == b.shape and not d1.any() and not d2.any()


GRAPHS = {   # edges of a frame graph: both directions, one, twice the same, a frame with itself
    "pairs": ([0, 1, 1, 2, 0, 2, 3, 2], [1, 0, 2, 1, 2, 0, 2, 3]),
    "mixed": ([0, 1, 0, 1, 2, 2, 3, 0, 1], [1, 0, 1, 2, 2, 2, 0, 0, 3]),
    "loops": ([1, 1, 2], [1, 1, 2])}


@pytest.mark.parametrize("K", [0, 5, 64])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("graph", list(GRAPHS))
@pytest.mark.parametrize("P,D,amp", [(190, 128, 1.0), (70, 40, 1.0), (129, 200, 1.0), (130, 128, 5.0), (65, 128, 0.0)])
def test_frame_graph_with_positive_gradients(P, D, amp, graph, dtype, K):
    """The gradient of a mean or a weighted sum: g >= 0, some of it 0 or tiny;
    amp 5: the rows' sums lie further apart than one exponential may serve;
    amp 0: all logits equal."""
    dt = TYPES[dtype]
    a, _, _, _, _, _, _ = _problem(P + D, dt, 0, 1, 4, P, 4, P, D, amp, shared=True)
    f1, f2 = (np.array(v, np.int32) for v in GRAPHS[graph])
    E = len(f1)
    _, _, _, _, idx, logits, g = _problem(P, dt, K, E, 4, P, 4, P, D, shared=True)
    g = np.abs(g)
    g[:, ::7] = 0.0
    g[:, 1::9] *= 1e-6
    p = (a, a, f1, f2, idx, logits, g)
    loss, grads = _run(*p, True, 1 / 16, 1.0)
    _check(dt, *p, True, 1 / 16, 1.0, loss, grads, PAIR)


def test_pairs_whose_one_side_is_dead_or_wrong():
    """An edge without a target, an edge out of range and left-out rows that are
    not finite, each with a live reverse."""
    dt = torch.float16
    a, _, _, _, idx, logits, g = _problem(21, dt, 3, 6, 4, 150, 4, 150, 64, shared=True)
    g = np.abs(g)
    f1, f2 = np.array([0, 1, 0, 2, 1, 3], np.int32), np.array([1, 0, 2, 0, 3, 1], np.int32)
    idx[1] = -1                               # (1, 0) has no target
    loss, grads = _run(a, a, f1, f2, idx, logits, g, True, 1 / 16, 1.0)
    _check(dt, a, a, f1, f2, idx, logits, g, True, 1 / 16, 1.0, loss, grads, PAIR)
    h1 = f1.copy()
    h1[5] = 4                                 # (3, 1) becomes an edge of a frame that is not there
    loss, grads = _run(a, a, h1, f2, idx, logits, g, True, 1 / 16, 1.0)
    on = torch.from_numpy((idx[5] >= 0).any(-1)).to(DEV)   # left-out rows: loss 0 there too
    assert torch.equal(loss[5].isnan(), on) and not loss[:5].isnan().any()
    assert not grads[0][[0, 2]].isnan().any()
    # frame 3's rows 5..9 have no target in their own edge, and are no key of a live edge
    b = a.clone()
    b[3, 5:10] = float("nan")
    idx[5, 5:10], idx[4] = -1, -1
    loss, grads = _run(b, b, f1, f2, idx, logits, g, True, 1 / 16, 1.0)
    b[3, 5:10] = 0.0
    _check(dt, b, b, f1, f2, idx, logits, g, True, 1 / 16, 1.0, loss, grads, PAIR)


def test_one_bad_row_of_a_pair():
    """A row whose target is out of range is NaN in both of its gradients and
    leaves the other frames alone."""
    dt = torch.bfloat16
    a, _, _, _, idx, _, g = _problem(22, dt, 0, 3, 3, 70, 3, 70, 32, shared=True)
    f1, f2 = np.array([0, 1, 2], np.int32), np.array([1, 0, 2], np.int32)
    idx[0, :, 0] = -1
    idx[0, 7, 0] = 70
    idx[1, :, 0] = np.where(np.arange(70) == 3, -1, 5)
    loss, grads = _run(a, a, f1, f2, idx, None, np.abs(g), True, 1 / 16, 1.0)
    assert loss[0, 7].isnan() and loss.isnan().sum() == 1
    assert grads[0][0, 7].isnan().all() and not grads[0][2].isnan().any()


@pytest.mark.parametrize("K", [0, 3])
@pytest.mark.parametrize("sign", [False, True])
def test_many_edges(sign, K):
    """More edges than one pass over the edge list holds, most of them paired."""
    dt = torch.float16
    p = list(_problem(23, dt, K, 700, 6, 70, 6, 70, 32, shared=True))
    if not sign:
        p[-1] = np.abs(p[-1])
    loss, grads = _run(*p, True, 1 / 16, 1.0)
    _check(dt, *p, True, 1 / 16, 1.0, loss, grads, PAIR)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_many_frames(dtype):
    """More frames than the plan's workgroup has threads, few of them used."""
    dt = TYPES[dtype]
    p = list(_problem(24, dt, 0, 40, 1500, 9, 1100, 12, 16))
    loss, grads = _run(*p, False, 1 / 16, 1.0)
    _check(dt, *p, False, 1 / 16, 1.0, loss, grads)
    unused = np.setdiff1d(np.arange(1500), p[2])
    assert not grads[0][torch.from_numpy(unused).to(DEV)].any()


@pytest.mark.parametrize("P,Q,K", [(130, 9000, 0), (9000, 130, 0), (70, 9000, 5), (9000, 70, 5)])
def test_long_frames(P, Q, K):
    """Frames longer than the streamed range whose sparse terms are sorted at once."""
    dt = torch.bfloat16
    p = list(_problem(25, dt, K, 2, 1, P, 2, Q, 8))
    loss, grads = _run(*p, False, 1 / 16, 1.0)
    _check(dt, *p, False, 1 / 16, 1.0, loss, grads)


def test_long_frames_both_ways():
    dt = torch.float16
    a, _, _, _, _, _, _ = _problem(26, dt, 0, 1, 2, 8300, 2, 8300, 8, shared=True)
    rng = np.random.default_rng(26)
    idx = rng.integers(-1, 8300, (2, 8300, 1)).astype(np.int32)
    f1, f2 = np.array([0, 1], np.int32), np.array([1, 0], np.int32)
    g = rng.random((2, 8300)).astype(np.float32)
    loss, grads = _run(a, a, f1, f2, idx, None, g, True, 1 / 16, 1.0)
    _check(dt, a, a, f1, f2, idx, None, g, True, 1 / 16, 1.0, loss, grads, PAIR)


@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_many_targets_on_few_keys(dtype, positive):
    """64 targets a row, all rows the same 64 keys and some keys twice: more
    sparse terms at one place than are kept in shared memory."""
    dt = TYPES[dtype]
    a, _, f1, f2, idx, logits, g = _problem(27, dt, 64, 3, 2, 700, 2, 700, 64, shared=True)
    f1[:], f2[:] = [0, 1, 0], [1, 0, 0]
    idx[:] = np.arange(64)
    idx[:, :, 60:] = 3
    idx[:, ::5, 10:20] = -1
    if positive:
        g = np.abs(g)
    p = (a, a, f1, f2, idx, logits, g)
    loss, grads = _run(*p, True, 1 / 16, 1.0)
    _check(dt, *p, True, 1 / 16, 1.0, loss, grads, PAIR)


def test_a_key_named_often_is_added_in_one_order():
    """Every row names three keys twenty times each with weights far apart:
    equal bits in every run."""
    import droid_backends as nb
    a, _, f1, f2, idx, logits, g = _problem(28, torch.float16, 60, 4, 2, 130, 2, 130, 64, shared=True)
    f1[:], f2[:] = [0, 1, 0, 1], [1, 0, 0, 1]
    idx[:] = (np.arange(60) % 3) * 40 + np.arange(130)[:, None] % 7
    k = (a, None, _t(f1), _t(f2), _t(idx))
    first = None
    for _ in range(4):
        loss, lse, prob = nb.corr_loss_forward(*k, _t(logits))
        d, _ = nb.corr_loss_backward(_t(np.abs(g)), *k, lse, prob)
        if first is None:
            first = (loss, prob, d)
        assert all(torch.equal(p, q) for p, q in zip(first, (loss, prob, d)))
    assert (prob[..., :3] > 0).any() and not prob[..., 3:].any()
    p = (a, a, f1, f2, idx, logits, np.abs(g))
    _check(torch.float16, *p, True, 1 / 16, 1.0, loss, [d], PAIR)


def test_offsets_past_32_bits():
    """2.6e9 feature values: the last two frames' edges as with these frames alone."""
    from droid_mi355x import corr_cross_entropy
    P, D, N = 65536, 128, 310
    g = torch.Generator(device=DEV).manual_seed(0)
    two = torch.randn((2, P, D), generator=g, device=DEV).bfloat16()
    t = torch.randint(0, P, (2, P), generator=g, device=DEV, dtype=torch.int32)
    t[:, ::3] = -1
    up = torch.rand((2, P), generator=g, device=DEV)
    many = torch.zeros((N, P, D), dtype=torch.bfloat16, device=DEV)
    many[-2:] = two
    out = []
    for x in (two, many):
        x = x.requires_grad_()
        k = x.shape[0] - 2
        f1, f2 = _t(np.array([k, k + 1], np.int32)), _t(np.array([k + 1, k], np.int32))
        loss = corr_cross_entropy(x, None, f1, f2, t)
        out.append((loss.detach(), torch.autograd.grad(loss, [x], up)[0]))
    assert torch.equal(out[0][0], out[1][0])
    d, e = out[0][1].float(), out[1][1][-2:].float()
    # the same sums in shares that may be cut elsewhere: a rounding to bf16 each
    assert ((d - e).abs() <= 2.0 ** -7 * d.abs() + 1e-6 * d.abs().max()).all()
    assert not out[1][1][:-2].any()
