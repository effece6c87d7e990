"""The scratch of a captured tree attention stays the graph's own when a larger call replaces it in its Workspace."""
import random

import pytest
import torch


def test_scratch_that_a_capture_was_given_is_kept():
    from nanoslg_amd import kernels
    ws = kernels.Workspace(torch.device("cpu"))
    got = []
    # (bytes, inside a capture): the second grows inside one, what the fourth made none was given
    for nbytes, capturing in ((1000, False), (3000, True), (2000, False), (9000, False), (20000, False), (20000, True), (40000, True),
                              (80000, False)):
        ws._capturing = lambda: capturing
        got.append(ws.get_prefill(nbytes))
        assert got[-1].numel() >= nbytes and got[-1] is ws.prefill_buf
    kept = [next(i for i, g in enumerate(got) if g is b) for b in ws._prefill_kept]
    assert kept == [0, 1, 4, 6] and got[1] is got[2] and got[4] is got[5]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_captured_tree_attention_keeps_its_scratch(dtype):
    """Two graphs with one workspace, the second of larger trees, and a larger eager call: the first graph's replays are its
    eager call's and leave tensors made since as they are."""
    from nanoslg_amd import kernels
    from test_gpu_tree import DEV, Setup, random_tree
    rng = random.Random(3)
    small, large, larger = (Setup(n, [c, 300], [random_tree(rng, n), random_tree(rng, 3)], dtype, 16, 8)
                            for n, c in ((9, 400), (60, 2000), (200, 9000)))
    ws = kernels.Workspace(torch.device(DEV))
    wants = [s.run() for s in (small, large, larger)]
    small.run(workspace=ws)
    torch.cuda.synchronize()
    graphs, outs, used = [], [], []
    for s in (small, large):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(s.run(workspace=ws))
        used.append((ws.prefill_buf.data_ptr(), ws.prefill_buf.data_ptr() + ws.prefill_buf.numel()))
    assert torch.equal(larger.run(workspace=ws), wants[2])
    used.append((ws.prefill_buf.data_ptr(), ws.prefill_buf.data_ptr() + ws.prefill_buf.numel()))
    used.sort()
    assert len({a for a, _ in used}) == 3 and all(a[1] <= b[0] for a, b in zip(used, used[1:]))
    others = [torch.zeros(b - a, dtype=torch.uint8, device=DEV) for a, b in used]  # (what the allocator has of these sizes)
    for _ in range(3):
        for i in (0, 1):
            outs[i].zero_()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], wants[i])
        assert torch.equal(larger.run(workspace=ws), wants[2])
        assert not any(o.any() for o in others)
