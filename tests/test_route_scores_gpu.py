"""fw_route_scores against a plain 64-bit implementation: the selection has to
be equal index for index, ties and near ties included; the weights are held
to bounds of f32 arithmetic."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import firewing_b200 as fw  # noqa: E402

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# expf, the quotients, the renormalising sum of 32 terms at most (6 levels)
# and the scale: under 16 roundings of 2^-24
WEIGHT_TOL = 16 * 2.0 ** -24
# a softmax kept unnormalised has the row's sum in it: at most 32 terms per
# lane, 5 levels and the terms' own errors, 2^-18.3 in all
SOFTMAX_SUM_TOL = 2.0 ** -18


def route_row(z, bias, scoring, groups, top_groups, group_top, top_k, renormalize, scale):
    """One row, from the definition: (indices, weights) in Python numbers."""
    z = [float(v) for v in z]
    E = len(z)
    live = [e for e in range(E) if z[e] != -math.inf and (bias is None or bias[e] != -math.inf)]
    if not live:
        return [-1] * top_k, [0.0] * top_k
    if scoring == "softmax":
        high = max(z)
        mass = math.fsum(math.exp(v - high) for v in z)
        score = [math.exp(v - high) / mass for v in z]
    else:
        score = [1.0 / (1.0 + math.exp(-v)) if v > -700 else 0.0 for v in z]
    key = [score[e] + (0.0 if bias is None else float(bias[e])) for e in range(E)]
    if groups > 1:
        size = E // groups
        members = {}
        for e in live:
            members.setdefault(e // size, []).append(key[e])
        rank = sorted(members, key=lambda g: (-sum(sorted(members[g])[::-1][:group_top]), g))[:top_groups]
        live = [e for e in live if e // size in rank]
    live.sort(key=lambda e: (-(key[e] if bias is not None else z[e]), e))
    chosen = live[:top_k]
    # ratios of exp(z) survive where the scores themselves underflow
    if renormalize:
        if scoring == "softmax":
            ref = max(z[e] for e in chosen)
            w = [math.exp(z[e] - ref) for e in chosen]
        else:
            ref = min(0.0, max(z[e] for e in chosen))
            w = [math.exp(min(z[e], 0.0) - ref) / (1.0 + math.exp(-abs(z[e]))) for e in chosen]
        total = math.fsum(w)
        w = [v / total for v in w]
    else:
        w = [score[e] for e in chosen]
    fill = top_k - len(chosen)
    return chosen + [-1] * fill, [v * scale for v in w] + [0.0] * fill


def run(logits, top_k, counts=False, stream=None, **kw):
    T, E = logits.shape
    idx = torch.full((T, top_k), -7, device="cuda", dtype=torch.int32)
    w = torch.full((T, top_k), 7.0, device="cuda")
    n = torch.full((E,), 99, device="cuda", dtype=torch.int32) if counts else None
    fw.route_scores(logits, idx, w, counts=n, stream=stream, **kw)
    torch.cuda.synchronize()
    return idx.cpu().numpy(), w.cpu().numpy(), None if n is None else n.cpu().numpy()


def check(logits, top_k, scoring="softmax", bias=None, groups=1, top_groups=1, group_top=1, renormalize=True,
          scale=1.0):
    idx, w, n = run(logits, top_k, counts=True, scoring=scoring, bias=bias, groups=groups, top_groups=top_groups,
                    group_top=group_top, renormalize=renormalize, scale=scale)
    z = logits.double().cpu().numpy()
    b = None if bias is None else bias.double().cpu().numpy()
    tol = SOFTMAX_SUM_TOL if scoring == "softmax" and not renormalize else WEIGHT_TOL
    want_n = np.zeros(logits.shape[1], np.int32)
    for t in range(len(z)):
        ri, rw = route_row(z[t], b, scoring, groups, top_groups, group_top, top_k, renormalize, scale)
        assert list(idx[t]) == ri, t
        np.testing.assert_allclose(w[t], rw, rtol=tol, atol=2.0 ** -126)
        for e in ri:
            if e >= 0:
                want_n[e] += 1
    assert np.array_equal(n, want_n)


def normal(seed, *shape, std=1.5, dtype="f32"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(DTYPES[dtype])


SHAPES = [  # T, E, K, groups, top_groups, group_top
    (1, 1, 1, 1, 1, 1), (3, 7, 7, 1, 1, 1), (5, 8, 1, 8, 1, 2), (1, 512, 10, 8, 4, 2), (9, 160, 6, 8, 3, 1),
    (33, 256, 8, 8, 4, 2), (4, 96, 32, 3, 2, 2), (6, 1024, 32, 32, 7, 2), (2, 999, 31, 27, 5, 2), (7, 64, 2, 32, 1, 2),
    (130, 32, 4, 4, 4, 1), (3, 33, 32, 1, 1, 1), (2, 31, 31, 31, 31, 2), (5, 992, 16, 31, 16, 1),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_shapes_scores_and_types(shape, scoring, biased, dtype):
    T, E, K, G, TG, GT = shape
    z = normal(E + T, T, E, dtype=dtype)
    bias = normal(7, E, std=0.1) if biased else None
    check(z, K, scoring, bias, G, TG, GT, renormalize=(E % 2 == 0), scale=2.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [None, "zero", "steps"])
@pytest.mark.parametrize("groups", [(1, 1, 1), (8, 3, 2)])
def test_equal_logits_go_to_the_lowest_index(scoring, bias, groups):
    z = torch.zeros(3, 64, device="cuda")
    z[1] = torch.randint(-2, 3, (64,), generator=torch.Generator().manual_seed(1)).float()
    z[2, ::2] = -0.0
    b = {None: None, "zero": torch.zeros(64, device="cuda"), "steps": (torch.arange(64, device="cuda") % 3) * 0.25}[bias]
    check(z, 9, scoring, b, *groups)
    check(z, 32, scoring, b, *((1, 1, 1) if groups[0] == 1 else (8, 4, 2)))


def test_near_ties_are_those_of_exact_scores():
    # Neighbouring f32 logits in the sigmoid's flat parts: scores nearer than
    # an f32 step, in either order of index.
    rng = np.random.default_rng(2)
    base = np.float32([9.0, 12.0, 14.0, 0.5, -3.0, 16.5])
    z = np.zeros((40, 48), np.float32)
    for t in range(40):
        for i in range(48):
            v = base[rng.integers(len(base))]
            for _ in range(int(rng.integers(0, 3))):
                v = np.nextafter(v, np.float32(100))
            z[t, i] = v
    z = torch.from_numpy(z).cuda()
    zero = torch.zeros(48, device="cuda")
    for scoring in ("softmax", "sigmoid"):
        check(z, 12, scoring, zero)
        check(z, 12, scoring, zero, 6, 2, 2)
        check(z, 12, scoring, None, 6, 2, 2)
    check(z, 32, "sigmoid", zero)


def test_near_ties_between_different_scores_and_biases():
    # bias = c - sigmoid(z) rounded to f32: every key is within an f32 step of c
    z = normal(3, 16, 64)
    z[:] = z[:1]
    s = torch.sigmoid(z[0].double())
    for c in (0.75, 1.0, 3.0):
        bias = (c - s).float()
        check(z, 20, "sigmoid", bias)
        check(z, 8, "sigmoid", bias, 8, 3, 2)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups", [(1, 1, 1), (8, 2, 2)])
def test_masked_experts(scoring, biased, groups):
    z = normal(4, 12, 64)
    z[:, ::3] = -math.inf
    z[3] = -math.inf                      # nothing left
    z[4] = -math.inf
    z[4, 17] = 0.5                        # one left
    z[5, 8:] = -math.inf                  # one group left
    z[6] = torch.finfo(torch.float32).min  # the type's lowest value is a value
    z[7, :32] = torch.finfo(torch.float32).min
    bias = normal(5, 64, std=0.1) if biased else None
    if biased:
        bias[10] = -math.inf
    check(z, 10, scoring, bias, *groups)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_far_logits_keep_their_ratios(scoring):
    z = torch.tensor([[-200.0, -201.0, -300.0, -199.5], [80.0, 90.0, 120.0, 200.0], [-90.0, -88.0, -89.0, -104.0],
                      [0.0, -120.0, 30.0, -150.0]], device="cuda")
    check(z, 3, scoring)
    check(z, 2, scoring, torch.tensor([0.0, 5.0, 9.0, 0.0], device="cuda"))


def test_rows_without_defined_scores():
    z = normal(6, 6, 40)
    z[1, 3] = math.nan
    z[3, 0] = math.inf
    for scoring, bad in (("softmax", {1, 3}), ("sigmoid", {1})):
        for bias in (None, torch.zeros(40, device="cuda")):
            idx, w, n = run(z, 4, counts=True, scoring=scoring, bias=bias)
            for t in range(6):
                assert (set(idx[t]) == {-1}) == (t in bad)
                assert np.isnan(w[t]).all() == (t in bad)
            assert n.sum() == 4 * (6 - len(bad))
    bias = torch.zeros(40, device="cuda")
    bias[2] = math.nan
    idx, w, n = run(z, 4, counts=True, scoring="sigmoid", bias=bias)
    assert (idx == -1).all() and np.isnan(w).all() and n.sum() == 0


def test_strided_rows_and_rows_behind_the_last():
    store = normal(8, 20, 100)
    z = store[2:15:2, 3:68]
    check(z, 5, "sigmoid")
    idx = torch.full((9, 5), -7, device="cuda", dtype=torch.int32)
    w = torch.full((9, 5), 7.0, device="cuda")
    fw.route_scores(z, idx[:7], w[:7], scoring="sigmoid")
    torch.cuda.synchronize()
    assert (idx[7:] == -7).all() and (w[7:] == 7.0).all()


def test_counts_are_overwritten_and_empty_batches():
    z = normal(9, 5, 16)
    a = run(z, 3, counts=True, scoring="sigmoid")
    b = run(z, 3, counts=True, scoring="sigmoid")
    assert np.array_equal(a[2], b[2]) and a[2].sum() == 15
    assert run(z[:0], 3, counts=True, scoring="sigmoid")[2].sum() == 0


def test_streams_and_graphs():
    z = normal(10, 700, 256, dtype="bf16")
    bias = normal(11, 256, std=0.1)
    kw = dict(scoring="sigmoid", bias=bias, groups=8, top_groups=4, group_top=2)
    want = run(z, 8, counts=True, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = run(z, 8, counts=True, stream=side, **kw)
    assert all(np.array_equal(a, b) for a, b in zip(want, got))
    outs, graphs = [], []
    for rows in (z, z.flip(0).contiguous()):
        o = (torch.empty(700, 8, device="cuda", dtype=torch.int32), torch.empty(700, 8, device="cuda"),
             torch.empty(256, device="cuda", dtype=torch.int32))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            fw.route_scores(rows, o[0], o[1], counts=o[2], stream=torch.cuda.current_stream(), **kw)
        outs.append(o)
        graphs.append((g, rows))
    for _ in range(2):
        for g, _rows in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert np.array_equal(outs[0][0].cpu().numpy(), want[0])
    assert np.array_equal(outs[1][0].cpu().numpy(), want[0][::-1])
    assert np.array_equal(outs[1][1].cpu().numpy(), want[1][::-1])
    assert np.array_equal(outs[0][2].cpu().numpy(), want[2]) and np.array_equal(outs[1][2].cpu().numpy(), want[2])


def test_the_reference_route_is_the_plain_case():
    # fw_route_bf16 (src/decoder_layer.rs:278-307): same selection, the
    # weights its bf16 roundings
    z = normal(12, 50, 512, dtype="bf16")
    idx, w, _ = run(z, 10)
    ri = torch.empty(50, 10, device="cuda", dtype=torch.int32)
    rs = torch.empty(50, 10, device="cuda", dtype=torch.bfloat16)
    fw.route_bf16(z, 50, 512, 10, ri, rs)
    assert np.array_equal(idx, ri.cpu().numpy())
    np.testing.assert_allclose(w, rs.float().cpu().numpy(), rtol=2.0 ** -8 + SOFTMAX_SUM_TOL)


@pytest.mark.parametrize("shape", [(512, 8), (1024, 32), (128, 4), (160, 8), (256, 16), (96, 3), (40, 5), (8, 2), (1000, 2)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("group_top", [1, 2])
def test_groups_that_nearly_tie(shape, scoring, biased, group_top):
    """Groups with the same logits in other orders, but for a step of f32 in
    one of the two best of some: scores that f32 cannot tell apart."""
    E, G = shape
    size = E // G
    r = np.random.default_rng(E + group_top)
    rows, b = [], None
    for t in range(24):
        base = r.normal(size=size).astype(np.float32) * 1.5 + 2.0
        z = np.stack([base.copy() for _ in range(G)])
        for g in range(G):
            steps, at = int(r.integers(-2, 3)), int(np.argsort(-base)[min(int(r.integers(0, 2)), size - 1)])
            for _ in range(abs(steps)):
                z[g, at] = np.nextafter(z[g, at], np.float32(np.inf if steps > 0 else -np.inf))
            if not biased:
                z[g] = z[g][r.permutation(size)]
        rows.append(z.reshape(-1))
    if biased:  # the same for every group, so that the sums stay near
        b = torch.tensor(np.tile(r.normal(size=size).astype(np.float32) * 0.1, G), device="cuda")
    z = torch.tensor(np.stack(rows), device="cuda")
    top_groups = max(1, G // 2)
    check(z, min(6, top_groups * size), scoring=scoring, bias=b, groups=G, top_groups=top_groups, group_top=group_top)


@pytest.mark.parametrize("shape", [(512, 8), (160, 8), (1024, 4)])
@pytest.mark.parametrize("biased", [False, True])
def test_groups_of_equal_experts(shape, biased):
    """More experts at a group's best score than are looked at singly."""
    E, G = shape
    z = torch.ones(5, E, device="cuda")
    z[1] = 0.5
    z[2, ::2] = 2.0
    z[3, E // 2:] = 1.0 + 2.0 ** -23
    z[4, -1] = 3.0
    b = torch.full((E,), 0.25, device="cuda") if biased else None
    for group_top in (1, 2):
        check(z, 5, scoring="sigmoid", bias=b, groups=G, top_groups=2, group_top=group_top)


@pytest.mark.parametrize("shape", [(64, 32), (128, 4), (256, 8), (160, 8), (512, 8), (40, 5)])
@pytest.mark.parametrize("scoring,largest,noise", [("softmax", 4.0, 1e-4), ("softmax", 128.0, 1e-4),
                                                   ("sigmoid", 16.0, 1e-5), ("sigmoid", 128.0, 1e-5)])
def test_groups_whose_two_best_keys_cancel(shape, scoring, largest, noise):
    """A group's two best keys are b + s and -b + s': their sum is small, its
    error in f32 that of b."""
    E, G = shape
    size = E // G
    r = np.random.default_rng(E)
    for _ in range(4):
        z = (0.3 + noise * r.normal(size=(40, E))).astype(np.float32)
        b = np.full((G, size), -1000.0, np.float32)
        b[:, 0] = r.uniform(largest / 2, largest, size=G)
        b[:, 1] = -b[:, 0]
        check(torch.tensor(z, device="cuda"), min(4, size), scoring=scoring, groups=G, top_groups=max(1, G // 2),
              group_top=2, bias=torch.tensor(b.reshape(-1), device="cuda"))


@pytest.mark.parametrize("shape", [(64, 8), (128, 4), (40, 5)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_groups_masked_by_the_lowest_value(shape, scoring):
    """Two keys near f32's lowest value add up to less than it; they are still
    ahead of a group without experts, and have an order."""
    E, G = shape
    size = E // G
    low = torch.finfo(torch.float32).min
    z = normal(30, 6, E)
    z[:, :size] = -math.inf  # the first group: nobody
    z[5, size:2 * size] = -math.inf
    for masks in ((low, low, 0.0), (low, 0.75 * low, 0.0), (0.75 * low, low, 0.6 * low), (low, low, low)):
        b = torch.zeros(G, size, device="cuda")
        b[1:] = masks[2]
        for g, m in enumerate(masks):
            b[1 + g] = m
        for top_groups in range(1, G + 1):
            for group_top in (1, 2):
                check(z, min(6, size), scoring=scoring, bias=b.reshape(-1).contiguous(), groups=G, top_groups=top_groups,
                      group_top=group_top)
    high = torch.finfo(torch.float32).max
    b = torch.zeros(G, size, device="cuda")
    b[1:] = high
    b[2] = 0.75 * high
    for top_groups in range(1, G + 1):
        check(z, min(6, size), scoring=scoring, bias=b.reshape(-1).contiguous(), groups=G, top_groups=top_groups,
              group_top=2)
