"""fw_token_logprobs against a plain 64-bit implementation."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import firewing_b200 as fw  # noqa: E402

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 2.0 ** -24


def sum_tol(vocab):
    """Relative error of the row's sums: a thread adds vocab / 256 terms in
    order, under 64 joins follow, and a term's own error is below 2^-21."""
    return (vocab / 256 + 64) * EPS + 2.0 ** -21


def normal(seed, *shape, std=2.5, dtype="bf16"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(DTYPES[dtype])


def run(z, targets=None, top_k=0, entropy=True, **kw):
    T = z.shape[0]
    lp = None if targets is None else torch.full(targets.shape, 7.0, device="cuda")
    h = torch.full((T,), 7.0, device="cuda") if entropy else None
    ti = torch.full((T, top_k), -7, device="cuda", dtype=torch.int32) if top_k else None
    tl = torch.full((T, top_k), 7.0, device="cuda") if top_k else None
    fw.token_logprobs(z, targets, lp, entropy=h, top_idx=ti, top_logprobs=tl, **kw)
    torch.cuda.synchronize()
    return [None if o is None else o.cpu().numpy() for o in (lp, h, ti, tl)]


def check(z, top_k=0, targets=None, temperature=1.0, seed=0):
    T, V = z.shape
    if targets is None:
        g = torch.Generator(device="cuda").manual_seed(seed)
        targets = torch.randint(0, V, (T, 3), generator=g, device="cuda", dtype=torch.int32)
    lp, h, ti, tl = run(z, targets, top_k, temperature=temperature)
    zz = z.double().cpu().numpy()
    ids = targets.cpu().numpy()
    s = sum_tol(V)
    for t in range(T):
        live = np.isfinite(zz[t])
        if not live.any():
            assert np.isneginf(lp[t]).all() and h[t] == 0.0
            assert top_k == 0 or ((ti[t] == -1).all() and np.isneginf(tl[t]).all())
            continue
        y = zz[t] / temperature
        m = y.max()
        p = np.exp(y - m)
        total = p.sum()
        want = y - m - math.log(total)
        with np.errstate(invalid="ignore"):
            want_h = -(p / total * np.where(p > 0, want, 0.0)).sum()
        # y itself: the logit's difference, log2(e) / temperature and their
        # product, four roundings
        np.testing.assert_allclose(lp[t], want[ids[t]], rtol=4 * EPS, atol=s + 4 * EPS * 64)
        # log2 S and W / S each up to log2(vocab)
        assert abs(h[t] - want_h) <= 3 * s * (math.log2(V) + 1)
        if top_k:
            order = np.lexsort((np.arange(V), -zz[t]))[:top_k]
            k = int(live[order].sum())
            assert list(ti[t][:k]) == list(order[:k]) and (ti[t][k:] == -1).all()
            np.testing.assert_allclose(tl[t][:k], want[order[:k]], rtol=4 * EPS, atol=s + 4 * EPS * 64)
            assert np.isneginf(tl[t][k:]).all()


@pytest.mark.parametrize("vocab", [1, 2, 5, 31, 255, 1000, 1025, 2047, 5003, 8192, 50021, 131072])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tokens", [1, 3])
def test_sizes_and_types(vocab, dtype, tokens):
    z = normal(vocab, tokens, vocab, dtype=dtype)
    for k in (0, 1, 5, 32):
        check(z, min(k, vocab))


@pytest.mark.parametrize("tokens", [17, 74, 150, 400])
def test_split_and_whole_rows(tokens):
    check(normal(tokens, tokens, 20001, dtype="f32"), 8)


def test_largest_vocabulary():
    check(normal(1, 2, 262144, dtype="bf16"), 20)
    check(normal(2, 1, 1 << 20, dtype="f32"), 32)


@pytest.mark.parametrize("temperature", [0.05, 0.7, 1.3, 30.0])
def test_temperature(temperature):
    check(normal(3, 5, 4099, dtype="f32"), 6, temperature=temperature)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [700, 5000, 40000])
def test_rows_that_fill_the_list(dtype, vocab):
    z = torch.zeros(6, vocab, device="cuda")
    z[1] = torch.arange(vocab, device="cuda") * 1e-3
    z[2] = -torch.arange(vocab, device="cuda") * 1e-3
    z[3] = (torch.arange(vocab, device="cuda") % 7).float()
    z[4, : vocab - 3] = -math.inf
    z[5, vocab // 2:] = 1.0
    z = z.to(DTYPES[dtype])
    for k in (1, 8, 31, 32):
        check(z, k)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_masks(dtype):
    V = 9001
    z = normal(4, 10, V, dtype=dtype)
    low = torch.finfo(DTYPES[dtype]).min
    z[0, ::2] = -math.inf
    z[1] = -math.inf
    z[2] = -math.inf
    z[2, 8000] = 3.0
    z[3, : V - 5] = -math.inf
    z[4] = low                   # the type's lowest value everywhere: a uniform row
    z[5, : V // 2] = low
    z[6] = low
    z[6, 17] = -100.0
    z[7, 5:] = -math.inf
    z[8] = -math.inf
    z[8, ::1000] = torch.finfo(DTYPES[dtype]).max / 2
    z[9, :3000] -= 200.0
    targets = torch.tensor([[0, 17, 8000, V - 1, 5]] * 10, device="cuda", dtype=torch.int32)
    check(z, 7, targets)


def test_sure_rows():
    # nearly all of the probability on one token, and on none of the first ones
    z = normal(5, 4, 30000, dtype="f32", std=1.0)
    z[0, 29999] = 40.0
    z[1, 0] = 90.0
    z[2, 15000] = 25.0
    z[3, 29000:] += 35.0
    check(z, 4)


def test_rows_with_nan_or_infinity():
    z = normal(6, 4, 3001, dtype="f32")
    z[1, 2000] = math.nan
    z[2, 5] = math.inf
    targets = torch.zeros(4, 1, device="cuda", dtype=torch.int32)
    lp, h, ti, tl = run(z, targets, 3)
    for t in range(4):
        bad = t in (1, 2)
        assert np.isnan(lp[t]).all() == bad and np.isnan(h[t]) == bad
        assert (ti[t] == -1).all() == bad and np.isnan(tl[t]).all() == bad
    big = torch.full((1, 40000), -math.inf, device="cuda")
    big[0, 39999] = math.nan  # in a part of its own, nothing else in the row
    lp, h, ti, tl = run(big, targets[:1], 3)
    assert np.isnan(lp).all() and np.isnan(h).all() and (ti == -1).all()


def test_targets_outside_the_vocabulary():
    z = normal(7, 2, 100)
    targets = torch.tensor([[-1, 3, 100], [5, -9, 2 ** 31 - 1]], device="cuda", dtype=torch.int32)
    lp = run(z, targets)[0]
    assert lp[0, 0] == 0.0 and lp[1, 1] == 0.0 and np.isnan(lp[0, 2]) and np.isnan(lp[1, 2])
    assert np.isfinite(lp[0, 1]) and np.isfinite(lp[1, 0])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shift", [0, 1, 3, 7])
def test_strided_and_unaligned_rows(dtype, shift):
    store = normal(8, 9, 4200, dtype=dtype)
    check(store[1:8:2, shift:shift + 4097], 5)
    check(store[:, shift:shift + 12], 5)


def test_offsets_past_32_bits():
    stride = (1 << 31) + 24
    store = torch.empty(stride + 1024, device="cuda", dtype=torch.bfloat16)
    z = torch.as_strided(store, (2, 1000), (stride, 1))
    z.copy_(normal(9, 2, 1000))
    check(z, 5)


def test_outputs_left_out_and_rows_behind_the_last():
    z = normal(10, 3, 6000)
    targets = torch.full((3, 2), 9, device="cuda", dtype=torch.int32)
    full = run(z, targets, 4)
    assert np.array_equal(run(z, targets, 0, entropy=False)[0], full[0])
    assert np.array_equal(run(z, None, 0)[1], full[1])
    only = run(z, None, 4, entropy=False)
    assert np.array_equal(only[2], full[2]) and np.array_equal(only[3], full[3])
    h = torch.full((5,), 7.0, device="cuda")
    fw.token_logprobs(z, entropy=h[:3])
    fw.token_logprobs(z[:0], entropy=h[:0])
    assert (h[3:] == 7.0).all()


def test_repeatable_on_streams_and_in_graphs():
    z = normal(11, 5, 70001, dtype="f32")
    targets = torch.randint(0, 70001, (5, 2), device="cuda", dtype=torch.int32)
    want = run(z, targets, 9)
    # the other order of rows, run eagerly: an odd row's place in memory decides
    # which values a thread adds up, so its sums are not those of another place
    flipped = run(z.flip(0).contiguous(), targets.flip(0).contiguous(), 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = run(z, targets, 9, stream=side)
    assert all(np.array_equal(a, b) for a, b in zip(want, got))
    outs, graphs = [], []
    for flip in (False, True):
        zz = z.flip(0).contiguous() if flip else z
        tt = targets.flip(0).contiguous() if flip else targets
        o = (torch.empty(5, 2, device="cuda"), torch.empty(5, device="cuda"),
             torch.empty(5, 9, device="cuda", dtype=torch.int32), torch.empty(5, 9, device="cuda"))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            fw.token_logprobs(zz, tt, o[0], entropy=o[1], top_idx=o[2], top_logprobs=o[3],
                              stream=torch.cuda.current_stream())
        outs.append(o)
        graphs.append((g, zz, tt))
    for _ in range(2):
        for g, *_ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for i in range(4):
        assert np.array_equal(outs[0][i].cpu().numpy(), want[i])
        assert np.array_equal(outs[1][i].cpu().numpy(), flipped[i])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("vocab", [2, 9, 54, 601, 5003, 50021])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_small_log_probabilities_keep_their_digits(dtype, vocab, temperature):
    """Where one token is nearly sure, log p and the entropy are small numbers:
    their relative errors are those of the other tokens' terms, a sum over
    vocab and a gap of up to 64 nats with four roundings."""
    tokens = 40
    z = normal(vocab, tokens, vocab, std=1.0, dtype=dtype).clamp_(-4, 4)
    at = (torch.arange(tokens, device="cuda") * 37 + (torch.arange(tokens, device="cuda") % 3 == 1) * (vocab - 1)) % vocab
    z[torch.arange(tokens, device="cuda"), at] = 16.0
    targets = at.to(torch.int32)[:, None].contiguous()
    for rows in (1, tokens):  # split rows and whole ones
        for top_k in (0, 2):
            lp, h, ti, tl = run(z[:rows], targets[:rows], top_k, temperature=temperature)
            y = z[:rows].double().cpu().numpy() / temperature
            p = np.exp(y - y.max(1, keepdims=True))
            ids = at[:rows].cpu().numpy()
            rest = np.where(np.arange(vocab)[None] == ids[:, None], 0.0, p).sum(1)
            tol = sum_tol(vocab) + 4 * EPS * 64
            np.testing.assert_allclose(lp[:, 0], -np.log1p(rest), rtol=tol)
            want = (y - y.max(1, keepdims=True)) - np.log1p(rest)[:, None]
            np.testing.assert_allclose(h, -(p / (1 + rest)[:, None] * want).sum(1), rtol=3 * tol)
            if top_k:
                assert (ti[:, 0] == ids).all() and (tl[:, 0] == lp[:, 0]).all()


def test_one_token_allowed():
    """Log p of the only token that a mask leaves is 0, and so is the entropy."""
    for vocab in (1, 7, 300, 40000):
        z = torch.full((5, vocab), -float("inf"), device="cuda", dtype=torch.bfloat16)
        at = torch.tensor([0, vocab - 1, vocab // 2, vocab // 3, vocab // 5], device="cuda")
        z[torch.arange(5, device="cuda"), at] = torch.tensor([3.3, -700.0, 0.1, 20000.0, -0.7], device="cuda").bfloat16()
        lp, h, ti, tl = run(z, at.to(torch.int32)[:, None].contiguous(), 1, temperature=0.7)
        assert (lp == 0).all() and (h == 0).all() and (tl == 0).all()
        assert (ti[:, 0] == at.cpu().numpy()).all()


def far_rows(seed, tokens, vocab, mask, dtype="f32"):
    """Rows filtered with a finite mask: in places, all but the last three, a
    first half, everything (a uniform row), all but one, a second half."""
    z = normal(seed, tokens, vocab, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    gone = torch.rand(tokens, vocab, generator=g, device="cuda") < 0.5
    at = torch.arange(vocab, device="cuda")
    for t in range(tokens):
        kind = t % 6
        if kind:
            gone[t] = (at < vocab - 3, at < vocab // 2, at >= 0, at != vocab // 3, at >= vocab // 2)[kind - 1]
    return z.masked_fill_(gone, mask)


@pytest.mark.parametrize("mask", [-1e8, -1e9, -1e10, -1.3e10, -1e11, -1e12, -1e20, -1e30])
@pytest.mark.parametrize("temperature", [1.0, 0.3, 0.1])
def test_rows_filtered_with_a_finite_mask(mask, temperature):
    for tokens, vocab in ((6, 50), (12, 5003), (6, 9001), (6, 131072)):
        check(far_rows(20, tokens, vocab, mask), 8, temperature=temperature)
    check(far_rows(21, 6, 5000, mask, "bf16"), 8, temperature=temperature)
    store = torch.full((6, 9100), mask, device="cuda")  # heads and tails that are no whole vectors
    store[:, 3:9004] = far_rows(22, 6, 9001, mask)
    check(store[:, 3:9004], 8, temperature=temperature)


def test_many_rows_filtered_with_a_finite_mask():
    check(far_rows(23, 450, 9001, -1e10), 8)
    check(far_rows(24, 450, 4096, -3e9), 8, temperature=0.3)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("size,temperature", [(6500.0, 1e-6), (30000.0, 1e-5), (1e4, 1e-4), (3.0, 1e-6), (50.0, 1e6),
                                              (1e10, 1.0), (1e11, 1.0), (1e9, 0.01), (1e12, 1e6)])
def test_far_logits_and_temperatures(dtype, size, temperature):
    if dtype == "f16" and size > 6e4:
        size = 6e4
    for tokens, vocab in ((3, 7), (5, 3001), (450, 9001), (4, 60000)):
        z = normal(25, tokens, vocab, std=1.0, dtype="f32").clamp_(-4, 4)
        z[0] = z[0].abs() * 0.2 * size + 0.1 * size  # every value far off on one side
        z[1] = -size - z[1].abs() * 2.0 ** -22 * size  # a few steps of f32 apart
        z[2:] *= size / 5
        check(z.to(DTYPES[dtype]), min(5, vocab), temperature=temperature)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("temperature", [3.0, 1e3, 1e6])
def test_differences_that_pass_the_largest_value(dtype, temperature):
    """Logits further apart than f32 holds, whose difference over the
    temperature is a number again."""
    high = torch.finfo(DTYPES[dtype]).max
    for vocab in (3, 5000, 40000):
        z = normal(26, 3, vocab, dtype=dtype)
        z[0, 0], z[0, 1] = high, -high
        z[1] = -high
        z[1, vocab // 2] = high
        z[2, 2] = 0.75 * high
        z[2, :2] = -0.5 * high
        targets = torch.tensor([[0, 1, vocab // 2, vocab - 1]] * 3, device="cuda", dtype=torch.int32)
        check(z, min(3, vocab), targets, temperature=temperature)
