"""Layers and clipping called from threads that run at the same time, and the reasons of refusals."""

import threading

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import test_gpu_expert_layers  # noqa: E402
import test_gpu_grad_clip  # noqa: E402
from test_gpu_expert_layers import block, block_inputs  # noqa: E402


@pytest.fixture(scope="module")
def ops():
    from lightgbm_rs_b200 import experts

    yield experts
    experts.check_errors()


@pytest.mark.parametrize("sizes", [(4000, 12, 136, 200, 72), (60, 40, 33, 129, 20)])
def test_threads_at_the_same_time(ops, sizes):
    """Threads that start together, each on a stream and inputs of its own: every step of every one
    has the bits that it has alone. A workspace or a sum shared between two calls would show in
    some step, whichever is spoiled."""
    count, steps = 4, 12
    inputs = [block_inputs(70 + i, *sizes) for i in range(count)]
    alone = [block(ops, *p, 1.0) for p in inputs]
    torch.cuda.synchronize()
    results, errors = [[] for _ in range(count)], []
    start = threading.Barrier(count)

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream), torch.no_grad():
                start.wait(60)
                for _ in range(steps):
                    results[i].append(block(ops, *inputs[i], 1.0))
            stream.synchronize()
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(count)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for got, want in zip(results, alone):
        assert len(got) == steps
        for step in got:
            assert all(torch.equal(a, b) for a, b in zip(step, want))


LAYERS = [
    "activation 'tanh'", "activation 2 ", r"bias: want \[2, 6\].*got \[2, 7\]",
    r"bias: want \[2, 6\].*got \[6\]", "bias: want .*got .*Float on", r"residual \[4, 7\].*want",
    r"residual \[5, 6\].*want", "residual .*Half on", "want a 2-D CUDA tensor.*cpu",
    "want a tensor of bfloat16 or float16", "x is 7 wide", "want w .*Half on",
    r"offsets: want \[3\].*got \[4\]", "offsets: want .*Long", "rows: want .*Long", "600 experts",
    "requires a gradient", "want gate and up", "activation 'swish'", "x is 9 wide",
    r"gradient \[4, 7\]", r"gradient \[5, 6\]", "gradient .*Half on", "want a torch tensor",
    r"pre: want \[4, 6\].*got \[4, 7\]", "pre: want .*got .*Half", "pre without an activation",
    "grad_dtype torch.float16", r"pre: want \[4, 2, 6\].*got \[4, 6\]",
    r"pre: want .*got \[4, 2, 7\]", r"gradient \[4, 12\]", "want gate and up",
    "grad_dtype torch.float64",
]
CLIP = [
    "no tensors", "got .*Double", "want CUDA tensors", "want a torch tensor", "max_norm -1",
    "max_norm nan", "0 results for 1", r"result 0 \[4\]", "result 0 .*Half", "overlaps another",
    "overlaps another", "overlaps another", "overlaps another", "overlaps another",
    "requires a gradient",
]


@pytest.mark.parametrize("file,i,message", [("layers", i, m) for i, m in enumerate(LAYERS)] +
                         [("clip", i, m) for i, m in enumerate(CLIP)])
def test_refused_for_its_own_reason(ops, file, i, message):
    from lightgbm_rs_b200 import LightGBMError

    calls = (test_gpu_expert_layers if file == "layers" else test_gpu_grad_clip).refusals()
    assert len(calls) == len(LAYERS if file == "layers" else CLIP)
    with pytest.raises(LightGBMError, match=message):
        calls[i](ops)
