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
    dict(counts=FAKE + 2), dict(dtype=0, logits=FAKE + 1)])
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
    dict(top_logprobs=FAKE + 3), dict(targets=0, top_k=0, entropy=None), dict(tokens=1 << 30)])
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
