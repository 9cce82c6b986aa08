"""examples/fp8_mlp.py: the block's four calls on weights that went through a
container give what the block gives in 64 bits, within 8-bit rounding, for one
token, a few and many, and under graph replay."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("fp8_mlp",
                                                  os.path.join(ROOT, "examples", "fp8_mlp.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.fixture(scope="module")
def block(example, tmp_path_factory):
    made = example.random_block(512, 1360, seed=3)
    path = str(tmp_path_factory.mktemp("mlp") / "mlp.tans.safetensors")
    made.save(path)
    loaded = example.Fp8Mlp.load(path)
    for name in ("norm", "gate_up", "gate_up_scale", "down", "down_scale"):
        assert torch.equal(getattr(loaded, name), getattr(made, name)), name
    return loaded


def _inputs(n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(n, 512, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2)]


@pytest.mark.parametrize("tokens", [1, 5, 33, 300, 1500])
def test_block_matches_64_bits(example, block, tokens):
    print(f"case: fp8 mlp {tokens} tokens", flush=True)
    x, res = _inputs(tokens, tokens)
    out = block.forward(x, res)
    want = example.reference(block, x, res)
    h = x.double() + res.double()
    # the branch alone: two roundings to 8 bits (relative 2-norm about 2^-5.2 each
    # for values spread over the format's binades) and two to bf16; the sum is
    # rounded to bf16 once more
    branch = (want - h).norm()
    assert (out.double() - want).norm() <= 2 * 2.0 ** -5 * branch + 2.0 ** -8 * want.norm()


def test_one_token_as_a_vector(block):
    x, res = _inputs(1, 9)
    assert torch.equal(block.forward(x[0], res[0]), block.forward(x, res)[0])


def test_block_in_a_graph(block):
    x, res = _inputs(7, 1)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        block.forward(x, res)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block.forward(x, res)
    for k in range(3):
        a, b = _inputs(7, 20 + k)
        x.copy_(a)
        res.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, block.forward(a, b))
