"""The example of the experts' operators that the package's guide gives, run as it stands there."""

import glob
import os
import re

import pytest
import torch

import dense_reference as R
import grouped_reference as G
from helpers import ROOT
from test_gpu_fp8 import _case
from test_gpu_grouped import DEV, _rand

pytestmark = pytest.mark.gpu


def _example():
    blocks = [b for path in sorted(glob.glob(os.path.join(ROOT, "*.md"))) for b in re.findall(r"```python\n(.*?)```", open(path).read(), re.S)
              if "api.fp8_gated_projection(" in b]
    assert len(blocks) == 1
    return compile(blocks[0], "example", "exec")


@pytest.mark.parametrize("tokens,top_k,ids_type", [(1, 2, torch.int64), (37, 3, torch.int32), (260, 2, torch.int64), (40, 1, torch.int32)])
def test_the_experts_of_the_guide(tokens, top_k, ids_type):
    """Every result is that of each route's own expert, the weighted sum that of each token's routes; eager, and captured with other routes at its replay."""
    from vllm_plugin_b200 import api
    experts, hidden, inter, channels = 6, 256, 144, 72
    x = _rand(1, tokens, hidden)
    w13, w2, w = _rand(2, experts, 2 * inter, hidden, std=0.1), _rand(3, experts, hidden, inter, std=0.1), _rand(4, experts, channels, hidden, std=0.1)
    _, _, w13_q, w13_scales = _case(1, experts, 2 * inter, hidden, 2)
    _, _, w2_q, w2_scales = _case(1, experts, hidden, inter, 1)
    w13_scales, w2_scales = w13_scales * 0.01, w2_scales * 0.01

    def routes(seed):
        weights, ids = torch.softmax(_rand(seed, tokens, experts, dtype=torch.float32), -1).topk(top_k, -1)
        return weights, ids.to(ids_type)

    topk_weights, topk_ids = routes(5)
    given = dict(torch=torch, api=api, x=x, topk_ids=topk_ids, topk_weights=topk_weights, top_k=top_k, E=experts, w13=w13, w2=w2, w=w, w13_q=w13_q,
                 w13_scales=w13_scales, w2_q=w2_q, w2_scales=w2_scales)
    example = _example()

    def check(got):
        flat = topk_ids.flatten().tolist()
        order = [r for e in range(experts) for r in range(len(flat)) if flat[r] == e]
        ends = torch.tensor([flat.count(e) for e in range(experts)]).cumsum(0).to(DEV)
        mine = x[torch.tensor([r // top_k for r in order], device=DEV)]
        block = G.Block(mine, w13, w2, ends, 10.0)
        R.check("y", got["y"], block.y, block.off["y"])
        one = G.Projection(mine, w, ends)
        R.check("p", got["p"], one.y, one.off["y"])
        # each token's sum of the routes' rows as they are, by FP32 weights: top_k products and additions
        want, size = torch.zeros(tokens, hidden, dtype=torch.float64, device=DEV), torch.zeros(tokens, hidden, dtype=torch.float64, device=DEV)
        for i, r in enumerate(order):
            add = got["y"][i].double() * topk_weights.flatten()[r].double()
            want[r // top_k] += add
            size[r // top_k] += add.abs()
        R.check("out", got["out"], want, 2 * top_k * 2.0 ** -24 * size + 2.0 ** -140)
        values, scales = G.quantize(mine)
        assert torch.equal(got["q"].double(), values) and torch.equal(got["s"], scales)
        R.check("h", got["h"], *G.fp8_product(got["q"], scales, w13_q, w13_scales, ends, torch.bfloat16, True, 10.0))
        values, scales = G.quantize(got["h"])
        R.check("z", got["z"], *G.fp8_product(values, scales, w2_q, w2_scales, ends, torch.bfloat16))
        api.read_dense_status()

    eager = dict(given)
    exec(example, eager)
    torch.cuda.synchronize()
    check(eager)
    captured = dict(given)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        exec(example, captured)
    for seed in (5, 6):
        weights, ids = routes(seed)
        topk_weights.copy_(weights)
        topk_ids.copy_(ids)
        graph.replay()
        torch.cuda.synchronize()
        check(captured)
