"""Refusals of the routing and log-probability primitives: decided before any
device call, so they need no GPU."""
import ctypes

import pytest

import firewing_b200 as fw
from firewing_b200 import moe

FAKE = 1 << 20  # an aligned address that nothing reads


def route(**kw):
    c = dict(experts=64, top_k=4, dtype=2, scoring=1, groups=8, top_groups=4, group_top=2, renormalize=1, scale=1.0,
             logit_stride=64)
    c.update({k: v for k, v in kw.items() if k in c})
    p = dict(logits=FAKE, tokens=1, bias=None, indices=FAKE, weights=FAKE, counts=None)
    p.update({k: v for k, v in kw.items() if k in p})
    return fw.library().fw_route_scores(ctypes.byref(moe._RouteConfig(**c)), p["logits"], p["tokens"], p["bias"],
                                        p["indices"], p["weights"], p["counts"], None)


@pytest.mark.parametrize("bad", [
    dict(experts=0), dict(experts=1025, logit_stride=1025), dict(top_k=0), dict(top_k=33), dict(groups=0),
    dict(groups=5), dict(groups=64), dict(top_groups=0), dict(top_groups=9), dict(group_top=0), dict(group_top=3),
    dict(top_groups=1, top_k=9), dict(scoring=2), dict(dtype=3), dict(dtype=-1), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(logit_stride=63), dict(tokens=-1), dict(logits=None), dict(indices=None),
    dict(weights=None), dict(logits=FAKE + 2), dict(bias=FAKE + 1), dict(indices=FAKE + 2), dict(weights=FAKE + 2),
    dict(counts=FAKE + 2), dict(dtype=0, logits=FAKE + 1), dict(tokens=(1 << 30) + 1), dict(logit_stride=1 << 38)])
def test_route_scores_refusals(bad):
    assert route(**bad) == fw.FW_EINVAL
    assert fw.library().fw_last_error()


def test_route_scores_without_tokens_is_a_success():
    assert route(tokens=0) == fw.FW_OK
    assert fw.library().fw_route_scores(None, FAKE, 1, None, FAKE, FAKE, None, None) == fw.FW_EINVAL


def logprobs(**kw):
    c = dict(vocab=100, dtype=0, targets=1, top_k=4, temperature=1.0, logit_stride=100)
    c.update({k: v for k, v in kw.items() if k in c})
    p = dict(logits=FAKE, tokens=1, ids=FAKE, logprobs=FAKE, entropy=FAKE, top_idx=FAKE, top_logprobs=FAKE)
    p.update({k: v for k, v in kw.items() if k in p})
    return fw.library().fw_token_logprobs(ctypes.byref(moe._LogprobConfig(**c)), *[p[k] for k in (
        "logits", "tokens", "ids", "logprobs", "entropy", "top_idx", "top_logprobs")], None)


@pytest.mark.parametrize("bad", [
    dict(vocab=0), dict(dtype=3), dict(targets=-1), dict(targets=65537), dict(top_k=-1), dict(top_k=33),
    dict(vocab=3), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
    dict(temperature=1e-7), dict(temperature=1e7), dict(logit_stride=99), dict(tokens=-1), dict(logits=None),
    dict(ids=None), dict(logprobs=None), dict(top_idx=None), dict(top_logprobs=None), dict(logits=FAKE + 1),
    dict(ids=FAKE + 2), dict(logprobs=FAKE + 2), dict(entropy=FAKE + 2), dict(top_idx=FAKE + 1),
    dict(top_logprobs=FAKE + 3), dict(targets=0, top_k=0, entropy=None), dict(tokens=1 << 30),
    dict(vocab=(1 << 30) + 1, logit_stride=1 << 31), dict(logit_stride=1 << 38)])
def test_token_logprobs_refusals(bad):
    assert logprobs(**bad) == fw.FW_EINVAL
    assert fw.library().fw_last_error()


def test_token_logprobs_without_tokens_is_a_success():
    assert logprobs(tokens=0) == fw.FW_OK


def test_the_bindings_take_tensors_of_one_gpu():
    torch = pytest.importorskip("torch")
    z = torch.zeros(2, 8)
    i = torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        fw.route_scores(z, i, torch.zeros(2, 2))
    with pytest.raises(ValueError, match="CUDA"):
        fw.token_logprobs(z, entropy=torch.zeros(2))
    with pytest.raises(ValueError, match="2-D"):
        fw.token_logprobs(z[0], entropy=torch.zeros(2))
    with pytest.raises(ValueError, match="scoring"):
        fw.route_scores(z, i, torch.zeros(2, 2), scoring="tanh")


def linear(**kw):
    c = dict(rows=64, cols=32, dtype=0, out_dtype=0, bias_dtype=2, residual_dtype=0, activation=0, w_stride=32,
             x_stride=32, residual_stride=64, y_stride=64)
    c.update({k: v for k, v in kw.items() if k in c})
    p = dict(w=FAKE, x=FAKE, tokens=1, bias=FAKE, residual=FAKE + 4096, y=FAKE)
    p.update({k: v for k, v in kw.items() if k in p})
    return fw.library().fw_linear_epilogue(ctypes.byref(moe._LinearConfig(**c)), *[p[k] for k in (
        "w", "x", "tokens", "bias", "residual", "y")], None)


@pytest.mark.parametrize("bad", [
    dict(rows=0), dict(cols=0), dict(rows=(1 << 24) + 1, residual_stride=1 << 25, y_stride=1 << 25),
    dict(cols=(1 << 24) + 1, w_stride=1 << 25, x_stride=1 << 25), dict(tokens=-1), dict(tokens=(1 << 24) + 1),
    dict(rows=1 << 20, tokens=1 << 20, residual_stride=1 << 20, y_stride=1 << 20), dict(dtype=2), dict(dtype=3),
    dict(out_dtype=1), dict(dtype=1), dict(bias_dtype=3), dict(residual_dtype=-1), dict(activation=-1),
    dict(activation=6), dict(w_stride=31), dict(x_stride=31), dict(residual_stride=63), dict(y_stride=63),
    dict(w_stride=1 << 38), dict(x_stride=1 << 38), dict(y_stride=1 << 38), dict(residual_stride=1 << 38),
    dict(w=None), dict(x=None), dict(y=None), dict(w=FAKE + 1), dict(x=FAKE + 1), dict(y=FAKE + 1),
    dict(out_dtype=2, y=FAKE + 2), dict(bias=FAKE + 2), dict(residual=FAKE + 1),
    dict(residual=FAKE, residual_dtype=2), dict(residual=FAKE, residual_stride=65)])
def test_linear_epilogue_refusals(bad):
    assert linear(**bad) == fw.FW_EINVAL
    assert fw.library().fw_last_error()


def test_linear_epilogue_without_tokens_is_a_success():
    assert linear(tokens=0) == fw.FW_OK


def test_the_linear_binding_takes_tensors_of_one_gpu():
    torch = pytest.importorskip("torch")
    w, x, y = (torch.zeros(4, 4, dtype=torch.bfloat16) for _ in range(3))
    with pytest.raises(ValueError, match="CUDA"):
        fw.linear_epilogue(w, x, y)
    with pytest.raises(ValueError, match="activation"):
        fw.linear_epilogue(w, x, y, activation="tanh")


@pytest.mark.parametrize("seconds", [0.0, 1e-6, 61.0])
def test_the_products_wait_limit_has_bounds(seconds):
    with pytest.raises(fw.FwError) as e:
        fw.primitive_set_wait_limit(seconds)
    assert e.value.code == fw.FW_EINVAL
    fw.primitive_set_wait_limit(2.0)


class Sized:
    """What the bindings look at before a call, of a tensor on the current GPU."""

    requires_grad = False

    def __init__(self, *shape, dtype):
        import torch

        self.shape, self.dtype, self.strides = torch.Size(shape), getattr(torch, dtype), [1]
        for n in shape[:0:-1]:
            self.strides.insert(0, self.strides[0] * n)

    def stride(self):
        return tuple(self.strides)

    def dim(self):
        return len(self.shape)

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return FAKE


BIG = (1 << 32) + 1  # one, to an int32


@pytest.fixture
def no_call(monkeypatch):
    pytest.importorskip("torch")
    monkeypatch.setattr(moe, "_call", lambda *a: pytest.fail("reached the library"))
    monkeypatch.setattr(moe, "_stream_of", lambda stream, device: 0, raising=False)


@pytest.mark.parametrize("T,N,K", [(BIG, 1, 1), (1, BIG, 1), (1, 1, BIG)])
def test_linear_sizes_beyond_the_interface_are_refused(no_call, T, N, K):
    w, x, y = Sized(N, K, dtype="bfloat16"), Sized(T, K, dtype="bfloat16"), Sized(T, N, dtype="bfloat16")
    with pytest.raises(ValueError, match="2\\^31"):
        fw.linear_epilogue(w, x, y)


@pytest.mark.parametrize("T,E,K", [(BIG, 4, 1), (1, BIG, 1), (1, 4, BIG)])
def test_route_sizes_beyond_the_interface_are_refused(no_call, T, E, K):
    with pytest.raises(ValueError, match="2\\^31"):
        fw.route_scores(Sized(T, E, dtype="float32"), Sized(T, K, dtype="int32"), Sized(T, K, dtype="float32"))


@pytest.mark.parametrize("name", ["groups", "top_groups", "group_top"])
@pytest.mark.parametrize("value", [BIG, 1 - (1 << 32)])
def test_route_numbers_beyond_the_interface_are_refused(no_call, name, value):
    with pytest.raises(ValueError, match="2\\^31"):
        fw.route_scores(Sized(2, 4, dtype="float32"), Sized(2, 1, dtype="int32"), Sized(2, 1, dtype="float32"),
                        **{name: value})


@pytest.mark.parametrize("T,V,C,K", [(BIG, 2, 1, 1), (1, BIG, 1, 1), (1, 2, BIG, 1), (1, 2, 1, BIG)])
def test_logprob_sizes_beyond_the_interface_are_refused(no_call, T, V, C, K):
    with pytest.raises(ValueError, match="2\\^31"):
        fw.token_logprobs(Sized(T, V, dtype="float32"), Sized(T, C, dtype="int32"), Sized(T, C, dtype="float32"),
                          top_idx=Sized(T, K, dtype="int32"), top_logprobs=Sized(T, K, dtype="float32"))


class Queue:
    """A torch.cuda.Stream, as far as the bindings look."""

    def __init__(self, device, handle=0):
        self.device_index, self.cuda_stream = device, handle


def three_operators(stream):
    h, f, i = "bfloat16", "float32", "int32"
    yield lambda: fw.linear_epilogue(Sized(4, 8, dtype=h), Sized(2, 8, dtype=h), Sized(2, 4, dtype=h), stream=stream)
    yield lambda: fw.route_scores(Sized(2, 4, dtype=f), Sized(2, 1, dtype=i), Sized(2, 1, dtype=f), stream=stream)
    yield lambda: fw.token_logprobs(Sized(2, 4, dtype=f), entropy=Sized(2, dtype=f), stream=stream)


@pytest.mark.parametrize("stream", [Queue(1), Queue(1, 77), "a name", object()])
def test_streams_of_another_device_and_other_objects_are_refused(monkeypatch, stream):
    # (a default stream's handle is 0 on every device)
    pytest.importorskip("torch")
    monkeypatch.setattr(moe, "_call", lambda *a: pytest.fail("reached the library"))
    for call in three_operators(stream):
        with pytest.raises(ValueError, match="stream"):
            call()


@pytest.mark.parametrize("stream,handle", [(Queue(0), 0), (Queue(0, 77), 77), (78, 78), (0, 0)])
def test_streams_that_are_given_are_passed_on(monkeypatch, stream, handle):
    pytest.importorskip("torch")
    seen = []
    monkeypatch.setattr(moe, "_call", lambda device, function, *args: seen.append((device, args[-1])))
    for call in three_operators(stream):
        call()
    assert seen == [(0, handle)] * 3


def test_tensors_that_require_a_gradient_are_refused(monkeypatch):
    """The outputs are written without autograd: a gradient would be lost."""
    torch = pytest.importorskip("torch")
    calls = []
    monkeypatch.setattr(moe, "_call", lambda *a: calls.append(a))
    h, f, i = "bfloat16", "float32", "int32"
    w, x, y, bias, residual = (Sized(4, 8, dtype=h), Sized(2, 8, dtype=h), Sized(2, 4, dtype=h), Sized(4, dtype=f),
                               Sized(2, 4, dtype=h))
    z, b, weights = Sized(2, 4, dtype=f), Sized(4, dtype=f), Sized(2, 1, dtype=f)
    logprobs, entropy = Sized(2, 1, dtype=f), Sized(2, dtype=f)

    def linear():
        fw.linear_epilogue(w, x, y, bias=bias, residual=residual, stream=0)

    def route():
        fw.route_scores(z, Sized(2, 1, dtype=i), weights, bias=b, stream=0)

    def logprob():
        fw.token_logprobs(z, Sized(2, 1, dtype=i), logprobs, entropy=entropy, stream=0)

    for call, tensors in ((linear, (w, x, y, bias, residual)), (route, (z, b, weights)), (logprob, (z, logprobs, entropy))):
        call()
        for t in tensors:
            t.requires_grad = True
            with pytest.raises(ValueError, match="gradient"):
                call()
            with torch.no_grad():
                call()
            t.requires_grad = False
    assert len(calls) == 3 + 11
