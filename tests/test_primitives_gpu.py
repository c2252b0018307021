"""What the dense product, the routing and the log probabilities have in
common: a first call inside a capture, calls of two streams at once, calls
from two threads."""
import os
import subprocess
import sys
import threading

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import firewing_b200 as fw  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FIRST = """
import torch, firewing_b200 as fw
torch.manual_seed(0)
w, x = torch.randn(512, 2048, device="cuda").bfloat16(), torch.randn({T}, 2048, device="cuda").bfloat16()
b = torch.zeros(512, device="cuda")
y = torch.empty({T}, 512, device="cuda")
i, v = torch.empty({T}, 8, device="cuda", dtype=torch.int32), torch.empty({T}, 8, device="cuda")
n = torch.empty(512, device="cuda", dtype=torch.int32)
h = torch.empty({T}, device="cuda")
torch.cuda.synchronize()
def run():
    s = torch.cuda.current_stream()
    fw.linear_epilogue(w, x, y, stream=s)
    fw.route_scores(y, i, v, scoring="sigmoid", bias=b, groups=8, top_groups=4, group_top=2, counts=n, stream=s)
    fw.token_logprobs(y, entropy=h, stream=s)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    run()
g.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (y, i, v, n, h)]
run()
torch.cuda.synchronize()
assert all(torch.equal(a, t) for a, t in zip(got, (y, i, v, n, h)))
assert n.sum().item() == 8 * {T}
"""


@pytest.mark.parametrize("T", [1, 64, 300])
def test_first_call_may_be_inside_a_capture(T):
    subprocess.run([sys.executable, "-c", FIRST.format(T=T)], check=True, cwd=ROOT, timeout=300)


def test_products_of_two_streams_at_once():
    # every kind of plan against every other, in flight together
    shapes = [(8, 2048, 2048), (64, 2048, 4096), (128, 2048, 2048), (256, 2048, 2048), (333, 1001, 1999),
              (700, 1024, 512), (2304, 2304, 512)]
    data = []
    for k, (T, N, K) in enumerate(shapes):
        g = torch.Generator(device="cuda").manual_seed(k)
        w = (torch.randn(N, K, generator=g, device="cuda") * K ** -0.5).bfloat16()
        x = torch.randn(T, K, generator=g, device="cuda").bfloat16()
        want = torch.empty(T, N, device="cuda", dtype=torch.bfloat16)
        fw.linear_epilogue(w, x, want, activation="silu")
        data.append((w, x, want))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for a in range(len(data)):
        for b in range(len(data)):
            outs = []
            for _ in range(6):
                for s, (w, x, want) in zip(streams, (data[a], data[b])):
                    y = torch.empty_like(want)
                    y.record_stream(s)
                    fw.linear_epilogue(w, x, y, activation="silu", stream=s)
                    outs.append((y, want))
            torch.cuda.synchronize()
            assert all(torch.equal(y, want) for y, want in outs)
    fw.primitive_status()


def test_two_threads():
    z = torch.randn(40, 30001, device="cuda")
    x, w = torch.randn(48, 1024, device="cuda").bfloat16(), torch.randn(700, 1024, device="cuda").bfloat16()

    def run(stream):
        h = torch.empty(40, device="cuda")
        i, p = torch.empty(40, 6, device="cuda", dtype=torch.int32), torch.empty(40, 6, device="cuda")
        y = torch.empty(48, 700, device="cuda")
        r, v = torch.empty(48, 8, device="cuda", dtype=torch.int32), torch.empty(48, 8, device="cuda")
        stream.wait_stream(torch.cuda.default_stream())
        fw.token_logprobs(z, entropy=h, top_idx=i, top_logprobs=p, stream=stream)
        fw.linear_epilogue(w, x, y, stream=stream)
        fw.route_scores(y, r, v, stream=stream)
        stream.synchronize()
        return h, i, p, y, r, v

    want = run(torch.cuda.Stream())
    failed = []

    def work():
        try:
            s = torch.cuda.Stream()
            for _ in range(20):
                if not all(torch.equal(a, b) for a, b in zip(run(s), want)):
                    failed.append("results")
        except Exception as e:  # noqa: BLE001
            failed.append(repr(e))

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    with pytest.raises(fw.FwError):
        fw.token_logprobs(z, entropy=want[0], temperature=0.0)


def three_calls(x, w, z, **kw):
    y = torch.zeros(48, 700, device="cuda")
    r, v = torch.zeros(48, 8, device="cuda", dtype=torch.int32), torch.zeros(48, 8, device="cuda")
    h = torch.zeros(40, device="cuda")
    fw.linear_epilogue(w, x, y, **kw)
    fw.route_scores(y, r, v, **kw)
    fw.token_logprobs(z, entropy=h, **kw)
    return y, r, v, h


def test_the_current_stream_is_the_default():
    w = torch.randn(700, 1024, device="cuda").bfloat16()
    x, z = torch.randn(48, 1024, device="cuda").bfloat16(), torch.randn(40, 30001, device="cuda")
    want = three_calls(x, w, z)
    torch.cuda.synchronize()
    # operands that the current stream writes late
    late_x, late_z = torch.zeros_like(x), torch.zeros_like(z)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(40_000_000)
        late_x.copy_(x)
        late_z.copy_(z)
        got = three_calls(late_x, w, late_z)
        fw.primitive_status()
        assert s.query()  # the stream that it waits for
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a stream that is given goes first
    with torch.cuda.stream(s):
        got = three_calls(x, w, z, stream=s.cuda_stream)
        s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # and so inside a capture
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = three_calls(x, w, z)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("K", [511, 1023, 999])
def test_a_chain_of_products_whose_rows_have_tails(K):
    """Each reads what the previous one has just written, from rows that are no
    whole words; their kernels overlap."""
    w = (torch.randn(K, K, device="cuda") * K ** -0.5).bfloat16()
    x = torch.randn(2, K, device="cuda").bfloat16()
    for T in (1, 2):
        chain = [x[:T].clone()] + [torch.zeros(T, K, device="cuda", dtype=torch.bfloat16) for _ in range(40)]
        single = [c.clone() for c in chain]
        torch.cuda.synchronize()
        for a, b in zip(single, single[1:]):
            fw.linear_epilogue(w, a, b)
            torch.cuda.synchronize()
        for a, b in zip(chain, chain[1:]):
            fw.linear_epilogue(w, a, b)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(chain, single))


def test_an_error_stays_with_its_call():
    """A call that CUDA refuses (here a wait inside a capture) says so itself and
    leaves nothing to the next one."""
    a = torch.randn(64, device="cuda").bfloat16()
    out = torch.empty_like(a)
    fw.linear_epilogue(a.view(1, 64), a.view(1, 64), torch.empty(1, 1, device="cuda"))
    fw.swiglu_bf16(a, a, 64, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(torch.cuda.Stream()):
        graph.capture_begin()
        with pytest.raises(fw.FwError, match="captur"):
            fw.primitive_status()
        with pytest.raises(RuntimeError):
            graph.capture_end()
    fw.swiglu_bf16(a, a, 64, out)
    fw.primitive_status()
