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


def test_an_error_on_one_stream_leaves_the_others_work_alone():
    """The workspaces are zeroed after a reported error: not while another stream's
    products, whose tiles CTAs hand to one another, are under way."""
    from flash_dllm_b200 import ops
    from flash_dllm_b200._lib import FdllmError, check_device_status
    g = tq._gen(5)
    a, sa = ops.quantize_int8(tq._randn(g, 64, 4096).bfloat16())
    w, sw = ops.quantize_int8(tq._randn(g, 4096, 4096).bfloat16())
    want = ops.linear_int8(a, sa, w, sw)
    q, caches, pt, spans, mb, tb, B, L = tq._attention_case(4, [(200, 1, 0), (150, 1, 0)], 2, 2, 200)
    tq._run_attention(q, caches, pt, mb, tb, B, L, 2, 2)
    bad = pt.clone()
    bad[0, 2] = 10 ** 6
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = [ops.linear_int8(a, sa, w, sw) for _ in range(400)]
    tq._run_attention(q, caches, bad, mb, tb, B, L, 2, 2)
    with pytest.raises(FdllmError):
        check_device_status()
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)
    out, sc = tq._run_attention(q, caches, pt, mb, tb, B, L, 2, 2)
    tq._check_attention(q, caches, pt, spans, B, L, 2, 2, out, sc)
