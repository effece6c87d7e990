"""Decode launchers kept over steps whose pages come and go: every plan that the workspace was sized for runs."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("batch,hq,hkv,d,page", [(192, 64, 8, 128, 16), (288, 48, 8, 128, 128), (400, 16, 2, 128, 16)])
@pytest.mark.parametrize("bits", [8, 16])
def test_a_launcher_rebound_to_plans_of_other_sizes(bits, batch, hq, hkv, d, page):
    """A workspace of exactly the bytes that the first plan's size asks for, then plans of up to its bound of pages."""
    from nanoslg_amd import kernels as K

    class Exact(K.Workspace):
        def get(self, nbytes):
            if self.buf.numel() < nbytes:
                self.buf = torch.zeros(nbytes, dtype=torch.uint8, device=DEV)
            return self.buf

    pools = [torch.zeros(1, batch + 2, page, hkv, d, dtype=torch.int8 if bits == 8 else torch.float16, device=DEV) for _ in "kv"]
    if bits == 8:
        pools += [torch.zeros(1, batch + 2, -(-page // 16), hkv, device=DEV) for _ in "kv"]
    q = torch.randn(batch, hq, d, device=DEV).half()
    row = torch.zeros(batch, hkv, d, device=DEV).half()

    def plan(pages):  # dealt out evenly; every sequence's last page its own, those before it one page of zeros
        n = np.full(batch, pages // batch) + (np.arange(batch) < pages % batch)
        ids = np.full(pages, batch + 1)
        ids[np.cumsum(n) - 1] = 1 + np.arange(batch)
        return i32((1 + np.arange(batch)) * page + page - 1), i32(np.concatenate([[0], np.cumsum(n)])), i32(ids), i32([page] * batch), pages

    launch = (K.DecodeLaunchQ8 if bits == 8 else K.DecodeLaunch)(*pools, *plan(batch), hq, workspace=Exact(torch.device(DEV)))
    for pages in (batch, 2 * batch, 528, 700, 900, 1024, 1050, 1100, 1150, 1200, 1265):
        if batch <= pages <= launch._ws_pages:
            launch.rebind(*plan(pages))
            assert not launch(0, q, row, row).any()
