"""The quantised operators on several streams at once, inside one captured graph."""
import pytest
import torch

import test_quantized_gpu as tq

pytestmark = pytest.mark.gpu
_no_device_error = tq._no_device_error


@pytest.mark.parametrize("rows", [8, 40])
def test_branches_of_one_captured_graph_keep_apart(rows):
    """Three streams that join one capture: products whose tiles CTAs share, key
    splits and column sums on each, all at the same time at a replay."""
    from flash_dllm_b200 import ops
    sts = [tq._step_state(41 + i, seqs=((512, 8, rows), (500, 8, 0), (450, 8, 3))) for i in range(3)]
    wants = [tq._step(ops, st) for st in sts]
    main, sides = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    outs = [None] * 3
    with torch.cuda.graph(graph, stream=main):
        for s in sides:
            s.wait_stream(main)
        for i, s in enumerate(sides):
            with torch.cuda.stream(s):
                outs[i] = tq._step(ops, sts[i])
        outs[2] = tq._step(ops, sts[2])
        # and again on every branch: a stream's calls follow one another
        for i, s in enumerate(sides):
            with torch.cuda.stream(s):
                outs[i] = tq._step(ops, sts[i])
        for s in sides:
            main.wait_stream(s)
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(outs, wants):
        for x, y in zip(got, want):
            assert torch.equal(x, y)
