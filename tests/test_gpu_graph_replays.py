"""Captured HIP graphs of what the package says can be captured: no memory-set nodes (replays after the first have read memory that such a node
had not cleared), and every replay equal to the eager result, with eager work in between."""
import os
import re

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _capture(fn, tmp_path):
    """(graph, what fn returned, the kinds of the graph's nodes)"""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    graph.enable_debug_mode()
    with torch.cuda.graph(graph):
        out = fn()
    path = os.path.join(tmp_path, "graph.dot")
    graph.debug_dump(path)
    with open(path) as f:
        text = f.read()
    kinds = {k: len(re.findall(r"\{\s*" + k, text)) for k in ("KERNEL", "MEMSET")}
    assert kinds["KERNEL"] > 0
    return graph, out, kinds


@pytest.mark.parametrize("views,rows", [(2, 256), (3, 256), (4, 256), (4, 7), (1, 33), (5, 4096)])
def test_attentive_aggregator_replays(tmp_path, views, rows):
    from mbvae_amd import blocks
    torch.manual_seed(views)
    net = blocks.AttentiveAggregator(1024, 1024, views, dropout=0.0).cuda().train()
    features = [torch.randn(rows, 1024, device="cuda", requires_grad=True) for _ in range(views)]
    weight = torch.randn(rows, 1024, device="cuda")
    leaves = [*features, *net.parameters()]

    def step():
        out, attn = net(features)
        return [out.detach(), attn.detach(), *torch.autograd.grad(out, leaves, weight)]

    graph, captured, nodes = _capture(step, tmp_path)
    assert nodes["MEMSET"] == 0, nodes
    for turn in range(4):
        if turn >= 2:                                        # (other values in the captured places)
            with torch.no_grad():
                for p in leaves:
                    p.mul_(0.9)
        want = [t.clone() for t in step()]
        for t in captured:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(captured, want)):
            assert torch.equal(a, b), f"replay {turn}, output {i}: {float((a - b).abs().max())}"


@pytest.mark.parametrize("fused", [False, True])
def test_encoder_train_step_with_adam_replays(tmp_path, fused):
    """A whole train step over encoders of the full width, their attentive aggregation and the fusion, with a capturable Adam: the losses of
    six replays are those of six eager steps (1e-3: Adam turns the rounding of a gradient that is zero in exact arithmetic into steps of its
    own; a gradient that is wrong moves the loss by half)."""
    from mbvae_amd import blocks, ops

    def make():
        torch.manual_seed(3)
        views = torch.nn.ModuleList([blocks.TransformerEncoder(d, 512, 1024, 2, dropout=0.0) for d in (256, 100, 1024)])
        return torch.nn.ModuleList([views, blocks.AttentiveAggregator(1024, 1024, 3, dropout=0.0),
                                    blocks.CrossAttentionFusion(1024, 64, 1, dropout=0.0)]).cuda().train()

    g = torch.Generator().manual_seed(4)
    inputs = [torch.randn(256, d, generator=g).cuda() for d in (256, 100, 1024)]
    target = torch.randn(256, 64, generator=g).cuda()

    def step(net, opt):
        views, aggregate, fuse = net
        a, _ = aggregate([enc(x) for enc, x in zip(views, inputs)])
        out = fuse(a, a.flip(0))
        loss = ((out[0] - target) ** 2).mean()
        loss.backward()
        opt.step()
        opt.zero_grad(set_to_none=True)
        return loss.detach()

    ops.set_fused_blocks(fused)
    try:
        losses = []
        for captured in (False, True):
            net = make()
            opt = torch.optim.AdamW(net.parameters(), lr=1e-3, fused=True, capturable=True)
            if not captured:
                losses.append([float(step(net, opt)) for _ in range(7)])
                continue
            first = []
            graph, loss, nodes = _capture(lambda: first.append(step(net, opt)) or first[-1], tmp_path)
            assert nodes["MEMSET"] == 0, nodes
            seen = [float(first[0])]
            for _ in range(6):
                graph.replay()
                torch.cuda.synchronize()
                seen.append(float(loss))
            losses.append(seen)
    finally:
        ops.set_fused_blocks(False)
    for k, (a, b) in enumerate(zip(*losses)):
        assert abs(a - b) <= 1e-3 * abs(a), f"step {k}: {losses}"
    assert abs(losses[0][-1] - losses[0][0]) > 1e-2 * abs(losses[0][0]), "the steps moved nothing"


@pytest.mark.parametrize("bs,low,high", [(3, 4, 20), (64, 10, 65), (300, 30, 65)])
def test_denoiser_inference_replays(tmp_path, bs, low, high):
    """The denoiser at its full widths over a ragged batch without gradients (the reverse step's network): the fused edge kernel takes its tasks
    from a counter that every call has to clear, also in a replay behind calls that have used it up."""
    from mbvae_amd.graph_transformer import GraphTransformer
    from mbvae_amd.trainstep import CFG3, synthetic_graphs
    torch.manual_seed(bs)
    net = GraphTransformer(**{**CFG3, "n_layers": 2}).cuda().eval()
    g = torch.Generator().manual_seed(bs)
    sizes = torch.randint(low, high, (bs,), generator=g)
    X0, E, mask = synthetic_graphs(bs, int(sizes.max()), "cuda", g, sizes=sizes)
    X = torch.cat((X0, torch.randn(bs, X0.shape[1], CFG3["input_dims"]["X"] - X0.shape[2], generator=g).cuda()), 2)
    y = torch.randn(bs, CFG3["input_dims"]["y"], generator=g).cuda()
    with torch.no_grad():
        net.prepare_padding_shortcuts(mask)

        def step():
            out = net(X, E, y, mask)
            return [out.X, out.E, out.y]

        graph, captured, nodes = _capture(step, tmp_path)
        assert nodes["MEMSET"] == 0, nodes
        for turn in range(4):
            X.mul_(0.9)
            y.neg_()
            want = [t.clone() for t in step()]
            for t in captured:
                t.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for k, a, b in zip("XEy", captured, want):
                assert torch.equal(a, b), f"replay {turn}, {k}"


@pytest.mark.parametrize("count", [7, 160, 161, 500])
def test_clipping_of_many_tensors_replays(tmp_path, count):
    """The table of the tensors, in the kernels' arguments or put together in the workspace, is part of the graph."""
    from mbvae_amd import ops
    g = torch.Generator().manual_seed(count)
    grads = [torch.randn(1 + (37 * i) % 900, generator=g).cuda() for i in range(count)]
    outs = [torch.empty_like(t) for t in grads]

    def step():
        return [ops.clip_grad_norm_(grads, 1.0, out=outs), *outs]

    graph, captured, nodes = _capture(step, tmp_path)
    assert nodes["MEMSET"] == 0, nodes
    for turn in range(4):
        for t in grads:
            t.mul_(-0.7)
        want = [t.clone() for t in step()]
        for t in captured:
            t.zero_()
        other = [torch.full((50,), 3.0, device="cuda") for _ in range(300)]           # (eager work that takes memory of its own)
        ops.clip_grad_norm_(other, 1.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(captured, want)):
            assert torch.equal(a, b), f"replay {turn}, output {i}"


@pytest.mark.parametrize("rows,V,D", [(4096, 5, 64), (4096, 700, 48), (40000, 3000, 24)])
def test_embedding_and_block_replay(tmp_path, rows, V, D):
    """Each route of the table's gradient, and the block's column sums, behind the first call of their kind or not."""
    from mbvae_amd import ops
    g = torch.Generator().manual_seed(rows + V)
    ids = torch.randint(-1, V, (rows,), generator=g).cuda()
    table = torch.randn(V, D, generator=g).cuda().requires_grad_(True)
    z = torch.randn(rows, D, generator=g).cuda().requires_grad_(True)
    gamma, beta = torch.rand(D, generator=g).cuda().requires_grad_(True), torch.randn(D, generator=g).cuda().requires_grad_(True)
    dy = torch.randn(rows, D, generator=g).cuda()

    def step():
        y, n = ops.gated_residual_norm(ops.embedding(ids, table), None, z, pre=(gamma, beta))
        return [y.detach(), n.detach(), *torch.autograd.grad([y, n], [table, z, gamma, beta], [dy, dy])]

    graph, captured, nodes = _capture(step, tmp_path)
    assert nodes["MEMSET"] == 0, nodes
    for turn in range(4):
        with torch.no_grad():
            ids.copy_(ids.flip(0))
            table.mul_(0.9)
        want = [t.clone() for t in step()]
        for t in captured:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(captured, want)):
            assert torch.equal(a, b), f"replay {turn}, output {i}"
