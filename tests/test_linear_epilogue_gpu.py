"""fw_linear_epilogue against a plain 64-bit implementation."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import firewing_b200 as fw  # noqa: E402

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid")


def normal(seed, *shape, std=1.0, dtype="bf16"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(DTYPES[dtype])


def reference(w, x, bias, activation, residual):
    """(result, bound of the f32 error before the final rounding)."""
    xd, wd = x.double(), w.double()
    v = xd @ wd.t()
    # Sums: every f32 addition errs by 2^-23 at most of the sum of magnitudes
    # (tensor cores may truncate), and a result has been through cols / 16 of
    # them on the tensor cores or cols / 256 plus a tree on the CUDA cores.
    size = xd.abs() @ wd.abs().t()
    err = (x.shape[1] / 16 + 16) * 2.0 ** -23 * size
    if bias is not None:
        v = v + bias.double()
        err = err + 2.0 ** -24 * v.abs()
    f = {"none": lambda a: a, "relu": lambda a: a.clamp(min=0),
         "gelu": lambda a: 0.5 * a * torch.special.erfc(-a * math.sqrt(0.5)),
         "gelu_tanh": lambda a: a / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3))),
         "silu": lambda a: a / (1 + torch.exp(-a)), "sigmoid": lambda a: 1 / (1 + torch.exp(-a))}[activation]
    if activation != "none":
        # slopes are below 1.13; the function's own error below 2^-20 of its
        # value while exponents stay under 16 in magnitude (2^-23.4 per unit)
        v = f(v)
        err = 1.13 * err + (2.0 ** -20 + 2.0 ** -16 * (activation != "relu")) * v.abs()
    if residual is not None:
        v = v + residual.double()
        err = err + 2.0 ** -24 * v.abs()
    return v, err


def check(w, x, y, bias=None, activation="none", residual=None, stream=None):
    want, err = reference(w, x, bias, activation, residual)
    fw.linear_epilogue(w, x, y, bias=bias, activation=activation, residual=residual, stream=stream)
    torch.cuda.synchronize()
    fw.primitive_status()
    half_step = torch.finfo(y.dtype).eps / 2
    tiny = torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    bound = err * (1 + half_step) + half_step * want.abs() + tiny
    off = (y.double() - want).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), int((off > bound).sum()), tuple(y.shape))


def case(T, N, K, dtype="bf16", out=None, activation="none", bias=None, residual=None, seed=0):
    w = normal(seed + 1, N, K, std=1 / math.sqrt(K), dtype=dtype)
    x = normal(seed + 2, T, K, dtype=dtype)
    b = None if bias is None else normal(seed + 3, N, dtype=bias)
    r = None if residual is None else normal(seed + 4, T, N, dtype=residual)
    y = torch.full((T, N), math.nan, device="cuda", dtype=DTYPES[out or dtype])
    check(w, x, y, b, activation, r)


# one token to many; K below, at and past a stage; one row; ragged edges
SIZES = [(1, 1, 1), (1, 512, 2048), (1, 7, 8192), (2, 33, 100), (3, 129, 64), (4, 1000, 257), (5, 1, 8), (5, 16, 16),
         (7, 130, 72), (16, 128, 64), (17, 129, 65), (33, 300, 1000), (64, 512, 2048), (96, 2048, 512),
         (127, 257, 129), (128, 128, 4096), (129, 128, 128), (130, 1, 64), (200, 1000, 136), (256, 256, 64),
         (300, 520, 8), (333, 1001, 1999), (513, 640, 320), (1000, 72, 1024), (2000, 2056, 256)]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
def test_sizes_and_types(size, dtype, out):
    case(*size, dtype=dtype, out=out, bias=dtype, residual=out)
    case(*size, dtype=dtype, out=out)


@pytest.mark.parametrize("size", [(2600, 2312, 200), (2304, 2304, 64), (4097, 4090, 136), (8192, 640, 1000),
                                  (20000, 264, 72)])
def test_many_tiles(size):
    case(*size, bias="bf16", activation="silu", residual="bf16")
    case(*size, dtype="f16", residual="f32")
    case(*size, out="f32", bias="f32")


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("size", [(1, 300, 512), (40, 300, 512), (300, 264, 512), (300, 263, 511)])
def test_activations(activation, size):
    for bias, residual in ((None, None), ("f32", None), (None, "bf16"), ("bf16", "f32")):
        case(*size, activation=activation, bias=bias, residual=residual)
    case(*size, dtype="f16", activation=activation, bias="f16", residual="f16")
    case(*size, out="f32", activation=activation, bias="f32", residual="f32")


@pytest.mark.parametrize("T", [1, 3, 40, 300])
@pytest.mark.parametrize("shift", [0, 1, 4, 8])
def test_strides_and_alignment(T, shift):
    N, K = 200, 328
    w = normal(1, N + 2, K + 40)[1:-1, shift:shift + K]
    x = normal(2, T + 2, K + 24)[1:-1, 8 - shift:8 - shift + K]
    r = normal(3, T, N + 11)[:, shift:shift + N]
    y = torch.full((T + 1, N + 16), 7.0, device="cuda", dtype=torch.bfloat16)
    check(w, x, y[:T, shift:shift + N], normal(4, N), "silu", r)
    assert bool((y[T:] == 7).all()) and bool((y[:, :shift] == 7).all()) and bool((y[:, shift + N:] == 7).all())
    odd = normal(5, T, 331)[:, :K]  # odd row stride
    check(w, odd, y[:T, shift:shift + N], normal(4, N), "none", r)


@pytest.mark.parametrize("T", [1, 4, 64, 300])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_residual_in_place(T, out):
    w, x = normal(1, 256, 512, std=0.05), normal(2, T, 512)
    y = normal(3, T, 256, dtype=out)
    want = y.clone()
    fresh = torch.empty_like(y)
    fw.linear_epilogue(w, x, fresh, activation="gelu", residual=want)
    fw.linear_epilogue(w, x, y, activation="gelu", residual=y)
    torch.cuda.synchronize()
    assert torch.equal(y, fresh)


def test_values_that_are_not_finite_stay_in_their_rows():
    for T in (2, 40, 300):
        w, x = normal(1, 144, 256, std=0.1), normal(2, T, 256)
        y, clean = (torch.empty(T, 144, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        fw.linear_epilogue(w, x, clean)
        x[1, 3] = math.nan
        w[5, 7] = math.inf
        fw.linear_epilogue(w, x, y, activation="relu")
        torch.cuda.synchronize()
        assert bool(torch.isnan(y[1]).all())
        rows = torch.ones(T, dtype=torch.bool, device="cuda")
        rows[1] = False
        cols = torch.ones(144, dtype=torch.bool, device="cuda")
        cols[5] = False
        assert torch.equal(y[rows][:, cols], clean[rows][:, cols].clamp(min=0))
        assert bool((torch.isinf(y[rows][:, 5]) | (y[rows][:, 5] == 0)).all())


def test_extreme_activations():
    v = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1.0, -1.0, 5.0, -5.0, 20.0, -20.0, 88.0, -88.0, 100.0, -100.0, 3e4,
                      -3e4, 1e30, -1e30], device="cuda").to(torch.bfloat16)
    w = v.view(-1, 1).contiguous()
    one = torch.ones(1, 1, device="cuda", dtype=torch.bfloat16)
    for T in (1, 8, 160):
        x = one.expand(T, 1).contiguous()
        for act, f in (("relu", lambda a: a.clamp(min=0)), ("gelu", torch.nn.functional.gelu),
                       ("gelu_tanh", lambda a: torch.nn.functional.gelu(a, approximate="tanh")),
                       ("silu", torch.nn.functional.silu), ("sigmoid", torch.sigmoid)):
            y = torch.empty(T, len(v), device="cuda")
            fw.linear_epilogue(w, x, y, activation=act)
            want = f(v.double()).expand(T, -1)
            torch.testing.assert_close(y.double(), want, rtol=2.0 ** -15, atol=2.0 ** -80 if act == "sigmoid" else 2.0 ** -75)


def test_offsets_past_32_bits():
    stride = (1 << 31) + 8
    store = torch.empty(2 * stride + 512, device="cuda", dtype=torch.bfloat16)
    for T, N in ((2, 3), (3, 40), (150, 3)):
        w = torch.as_strided(store, (3, 512), (stride, 1))
        w.copy_(normal(1, 3, 512, std=0.1))
        x = normal(2, T, 512)
        check(w, x, torch.empty(T, 3, device="cuda", dtype=torch.bfloat16))


def test_repeatable_on_streams_and_in_graphs():
    for T, N, K in ((1, 512, 2048), (64, 1024, 2048), (700, 512, 1024), (50, 333, 777)):
        w, b = normal(1, N, K, std=1 / math.sqrt(K)), normal(2, N)
        xs = [normal(3 + i, T, K) for i in range(2)]
        want = []
        for x in xs:
            y = torch.empty(T, N, device="cuda", dtype=torch.bfloat16)
            fw.linear_epilogue(w, x, y, bias=b, activation="silu")
            want.append(y)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = torch.empty_like(want[0])
        fw.linear_epilogue(w, xs[0], got, bias=b, activation="silu", stream=side)
        side.synchronize()
        assert torch.equal(got, want[0])
        outs, graphs = [], []
        for x in xs:
            y = torch.empty_like(want[0])
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                fw.linear_epilogue(w, x, y, bias=b, activation="silu", stream=torch.cuda.current_stream())
            outs.append(y)
            graphs.append(g)
        for _ in range(2):
            for g in graphs:
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_empty_batch_leaves_y():
    y = torch.full((3, 8), 7.0, device="cuda", dtype=torch.bfloat16)
    fw.linear_epilogue(normal(1, 8, 16), normal(2, 3, 16)[:0], y[:0])
    assert bool((y == 7).all())


def test_a_run_from_hidden_states_to_log_probabilities():
    """A gate and its routing, a dense layer on the residual stream, a head and
    its log probabilities, in one stream without a wait."""
    T, H, E, V = 20, 256, 64, 5000
    x = normal(1, T, H)
    gate, up, down, head = (normal(2 + i, n, k, std=1 / math.sqrt(k)) for i, (n, k) in enumerate(
        ((E, H), (2 * H, H), (H, 2 * H), (V, H))))
    bias = normal(8, E, std=0.1, dtype="f32")
    z = torch.empty(T, E, device="cuda")
    idx, wts = torch.empty(T, 6, device="cuda", dtype=torch.int32), torch.empty(T, 6, device="cuda")
    h, out = torch.empty(T, 2 * H, device="cuda", dtype=torch.bfloat16), x.clone()
    logits = torch.empty(T, V, device="cuda", dtype=torch.bfloat16)
    targets = torch.arange(T, device="cuda", dtype=torch.int32).view(T, 1)
    lp, ent = torch.empty(T, 1, device="cuda"), torch.empty(T, device="cuda")
    ti, tl = torch.empty(T, 4, device="cuda", dtype=torch.int32), torch.empty(T, 4, device="cuda")
    fw.linear_epilogue(gate, x, z)
    fw.route_scores(z, idx, wts, scoring="sigmoid", bias=bias, groups=8, top_groups=4, group_top=2)
    fw.linear_epilogue(up, x, h, activation="silu")
    fw.linear_epilogue(down, h, out, residual=out)
    fw.linear_epilogue(head, out, logits)
    fw.token_logprobs(logits, targets, lp, entropy=ent, top_idx=ti, top_logprobs=tl)
    torch.cuda.synchronize()
    # each step from the previous one's own output
    want, err = reference(gate, x, None, "none", None)
    assert bool(((z.double() - want).abs() <= err + 2.0 ** -24 * want.abs()).all())
    key = torch.sigmoid(z.double()) + bias.double()
    best = key.view(T, 8, 8).sort(2, descending=True).values[:, :, :2].sum(2).sort(1, descending=True).indices[:, :4]
    kept = torch.zeros(T, 8, dtype=torch.bool, device="cuda").scatter_(1, best, True).repeat_interleave(8, 1)
    order = key.masked_fill(~kept, -math.inf).sort(1, descending=True).indices[:, :6]
    assert torch.equal(order.int(), idx)
    s = torch.gather(torch.sigmoid(z.double()), 1, order)
    torch.testing.assert_close(wts.double(), s / s.sum(1, keepdim=True), rtol=2.0 ** -20, atol=0)
    for y, (ww, xx, act, res) in ((h, (up, x, "silu", None)), (out, (down, h, "none", x)),
                                  (logits, (head, out, "none", None))):
        want, err = reference(ww, xx, None, act, res)
        assert bool(((y.double() - want).abs() <= err * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()).all())
    q = torch.log_softmax(logits.double(), 1)
    torch.testing.assert_close(lp.double(), q.gather(1, targets.long()), rtol=0, atol=2.0 ** -15)
    torch.testing.assert_close(ent.double(), -(q.exp() * q).sum(1), rtol=0, atol=2.0 ** -12)
    torch.testing.assert_close(tl.double(), q.sort(1, descending=True).values[:, :4], rtol=0, atol=2.0 ** -15)


@pytest.mark.parametrize("tokens", [1, 5, 200, 600])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_activations_at_infinities_and_large_values(tokens, out):
    """Sums (here the bias alone) at the ends of the range: the limits of each
    activation, and NaN."""
    inf, nan = math.inf, math.nan
    at = [inf, -inf, nan, 3e38, -3e38, 1e25, -1e25, 200.0, -200.0, 0.0]
    limits = {
        "none": at,
        "relu": [inf, 0, nan, 3e38, 0, 1e25, 0, 200.0, 0, 0],
        "gelu": [inf, 0, nan, 3e38, 0, 1e25, 0, 200.0, 0, 0],
        "gelu_tanh": [inf, 0, nan, 3e38, 0, 1e25, 0, 200.0, 0, 0],
        "silu": [inf, 0, nan, 3e38, 0, 1e25, 0, 200.0, 0, 0],
        "sigmoid": [1, 0, nan, 1, 0, 1, 0, 1, 0, 0.5],
    }
    rows = 320
    x = torch.ones(tokens, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(rows, 64, device="cuda", dtype=torch.bfloat16)
    bias = torch.tensor(at * (rows // len(at)), device="cuda")
    for act, want in limits.items():
        y = torch.empty(tokens, rows, device="cuda", dtype=DTYPES[out])
        fw.linear_epilogue(w, x, y, bias=bias, activation=act)
        expected = torch.tensor(want * (rows // len(at)), device="cuda").expand(tokens, rows)
        if act != "sigmoid":
            expected = expected.to(y.dtype)  # one rounding; 200 and 0 are exact
        # (a sigmoid's quotient in f32: 2^-22)
        torch.testing.assert_close(y.float(), expected.float(), rtol=2.0 ** -22, atol=1e-30, equal_nan=True)


@pytest.mark.parametrize("size", [(5, 40, 9), (64, 129, 63), (100, 300, 1030), (112, 700, 517), (130, 2049, 333),
                                  (333, 1001, 1999), (1100, 1030, 2049), (2000, 3001, 257), (7000, 2060, 70)])
@pytest.mark.parametrize("out", ["f16", "f32"])
@pytest.mark.parametrize("shift", [(1, 3), (0, 2), (7, 0)])
def test_rows_at_odd_addresses_amid_nan(size, out, shift):
    """Operands whose rows start anywhere, with NaN between and around them."""
    T, N, K = size

    def amid(seed, rows, cols, at, pad, std=1.0):
        whole = torch.full((rows + 2, cols + pad), math.nan, device="cuda", dtype=torch.float16)
        whole[1:-1, at:at + cols] = normal(seed, rows, cols, std=std, dtype="f16")
        return whole[1:-1, at:at + cols]

    w = amid(1, N, K, shift[0], 11, std=1 / math.sqrt(K))
    x = amid(2, T, K, shift[1], 8)
    y = torch.full((T, N), math.nan, device="cuda", dtype=DTYPES[out])
    check(w, x, y, normal(3, N, dtype="f32"), "silu", normal(4, T, N, dtype="f16"))
    check(w, x, y)


@pytest.mark.parametrize("size", [(2600, 2312, 200), (4097, 4090, 136), (3000, 3000, 1032), (8192, 1600, 520), (2100, 8000, 64)])
def test_f32_outputs_of_many_tiles(size):
    case(*size, out="f32")
    case(*size, out="f32", bias="bf16", activation="gelu", residual="bf16")
    case(*size, dtype="f16", out="f32", activation="silu", residual="f32")
    T, N, K = size  # outputs and residual at odd addresses
    w, x = normal(1, N, K, std=1 / math.sqrt(K)), normal(2, T, K)
    y = torch.full((T + 1, N + 5), 7.0, device="cuda")
    check(w, x, y[:T, 3:3 + N], normal(3, N), "none", normal(4, T, N + 1)[:, 1:])
    assert bool((y[T:] == 7).all()) and bool((y[:, :3] == 7).all()) and bool((y[:, 3 + N:] == 7).all())


@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_the_wait_limit_bounds_steps_and_not_the_product(out):
    """A product that takes several times the limit of its waits (14 ms at the
    least for 2.3e13 operations; pairs of CTAs)."""
    T, N, K = 16384, 22528, 32768
    w, x = normal(1, N, K, std=1 / math.sqrt(K)), normal(2, T, K)
    want, y = (torch.full((T, N), math.nan, device="cuda", dtype=DTYPES[out]) for _ in range(2))
    fw.linear_epilogue(w, x, want)
    torch.cuda.synchronize()
    fw.primitive_set_wait_limit(0.003)
    try:
        fw.linear_epilogue(w, x, y)
        torch.cuda.synchronize()
        fw.primitive_status()
    finally:
        fw.primitive_set_wait_limit(2.0)
    assert torch.equal(y, want)
    rows = torch.arange(0, T, T // 64, device="cuda")
    part, err = reference(w, x[rows], None, "none", None)
    half_step = torch.finfo(y.dtype).eps / 2
    assert bool(((y[rows].double() - part).abs() <= err * (1 + half_step) + half_step * part.abs()).all())


@pytest.mark.parametrize("activation", ["gelu", "gelu_tanh", "silu", "sigmoid"])
@pytest.mark.parametrize("tokens", [1, 5, 200, 600])
def test_activations_keep_their_digits(activation, tokens):
    """f32 outputs of a sum v (the bias alone).  Each is a product with 2^e, e
    an f32 of size |e|: k roundings on its way cost ln 2 k 2^-24 |e|, and the
    rest is an exponential (2^-22), a reciprocal (2^-23), an addition and a
    product (2^-24 each): 2^-21.  k is 2 for SiLU and the sigmoid (log2 e and the
    product), 8 for the tanh form (the constants' five, v^2, a sum and a
    product), 3 for the erf form (v^2, its constant, a sum), whose polynomial
    adds nine roundings of sums up to 2 and its fit: 2^-20.  What is below f32's
    normal numbers times v's size (at most 88) may be 0."""
    k, fixed = {"silu": (2, 2.0 ** -21), "sigmoid": (2, 2.0 ** -21), "gelu_tanh": (8, 2.0 ** -21),
                "gelu": (3, 2.0 ** -21 + 2.0 ** -20)}[activation]
    rows = 4096
    v = torch.logspace(-6, 2, rows // 2, dtype=torch.float64, device="cuda").float()
    v = torch.cat((v, -v))
    x = torch.ones(tokens, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(rows, 64, device="cuda", dtype=torch.bfloat16)
    y = torch.empty(tokens, rows, device="cuda")
    fw.linear_epilogue(w, x, y, bias=v, activation=activation)
    a = v.double()
    cubic = math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)
    want, e = {"silu": (a / (1 + torch.exp(-a)), a), "sigmoid": (1 / (1 + torch.exp(-a)), a),
               "gelu_tanh": (a / (1 + torch.exp(-2 * cubic)), 2 * cubic),
               "gelu": (0.5 * a * torch.special.erfc(-a * math.sqrt(0.5)), 0.5 * a * a)}[activation]
    bound = (fixed + math.log(2.0) * k * 2.0 ** -24 * e.abs() / math.log(2.0)) * want.abs() * (1 + 2.0 ** -10)
    bound = bound.clamp(max=1e300) + 88 * 2.0 ** -126
    off = (y.double() - want).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), float(v[(off / bound).max(0).values.argmax()]))


def rms_error(T, N, K, x_shift=0, dtype="bf16"):
    w = normal(1, N, K + 1, std=1 / math.sqrt(K), dtype=dtype)[:, x_shift:K + x_shift]
    x = normal(2, T, K + 8, dtype=dtype)[:, :K]
    if not x_shift:
        w, x = w.contiguous(), x.contiguous()
    y = torch.full((T, N), math.nan, device="cuda")
    fw.linear_epilogue(w, x, y)
    want = x.double() @ w.double().t()
    return float(((y.double() - want).norm() / want.norm()))


# tiles shared by a cluster, tiles of a CTA alone (w and x on the M side), pairs of CTAs, loaders
@pytest.mark.parametrize("size,shift", [((64, 512, 65536), 0), ((24, 20000, 8192), 0), ((400, 20000, 8192), 0),
                                        ((1100, 640, 16384), 0), ((2304, 2304, 8192), 0), ((4096, 4096, 16384), 0),
                                        ((50, 20000, 8191), 1), ((700, 3001, 8191), 1)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_f32_outputs_of_long_sums(size, shift, dtype):
    """The tensor cores cut sums off, which one accumulation over 8192 columns
    shows: 1.4e-6 of the outputs, in pieces of 512 columns 4.4e-7 (measured).
    The limit between them is their geometric mean."""
    assert rms_error(*size, shift, dtype) <= 8e-7


@pytest.mark.parametrize("size", [(1, 300, 512), (40, 300, 512), (300, 264, 512), (2304, 2304, 128)])
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_a_bias_at_any_address(size, out, shift):
    """A slice of a fused parameter: the outputs are those of an aligned bias."""
    T, N, K = size
    w, x, r = normal(1, N, K, std=1 / math.sqrt(K)), normal(2, T, K), normal(3, T, N, dtype=out)
    for dtype in ("bf16", "f32"):
        store = normal(4, N + 8, dtype=dtype)
        bias = store[shift:shift + N]
        y, want = (torch.full((T, N), math.nan, device="cuda", dtype=DTYPES[out]) for _ in range(2))
        check(w, x, y, bias, "gelu", r)
        fw.linear_epilogue(w, x, want, bias=bias.clone(), activation="gelu", residual=r)
        assert torch.equal(y, want)
