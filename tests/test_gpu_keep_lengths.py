"""The lengths that flash_keep_paged returns do not depend on the caches: there may be no layers, or no pages."""
import pytest
import torch

import scored_reference as ref
from paged_reference import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("own_path", [False, True])
@pytest.mark.parametrize("what", ["layers", "pages", "layers and pages"])
def test_lengths_without_rows(fa, what, own_path):
    batch = Batch([6, 1, 0, 9], [30, 1, 16, 100], 2, 2, 64, 16, torch.float16, seed=2)
    path = torch.tensor([[0, 2, 3, 5], [0, -1, -1, -1], [-1, -1, -1, -1], [3, 2, 8, 8]], dtype=torch.int32)
    accepted = torch.tensor([4, 1, 0, 3], dtype=torch.int32)
    _, _, want = ref.keep(batch.k_cache, batch.v_cache, batch.table, batch.lens, batch.cu, path, accepted)
    assert want.tolist() == [28, 1, 16, 92]
    shape = [0 if "layers" in what else 2, 0 if "pages" in what else 12, 2, 16, 64]
    index = [t.cuda() for t in (batch.table, batch.lens, batch.cu, path, accepted)]
    caches = [torch.zeros(shape if "layers" in what else shape[1:], dtype=torch.float16, device="cuda") for _ in range(2)]
    how = {"stream": torch.cuda.current_stream()} if own_path else {}
    out = torch.full((4,), -77, dtype=torch.int32, device="cuda")
    assert fa.flash_keep_paged(*caches, *index, out=out, **how) is out
    assert torch.equal(out.cpu(), want)
    assert torch.equal(fa.flash_keep_paged(*caches, *index, **how).cpu(), want)


def test_no_sequences_no_layers(fa):
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    caches = [torch.zeros((0, 3, 2, 16, 64), dtype=torch.float16, device="cuda") for _ in range(2)]
    after = fa.flash_keep_paged(*caches, none.view(0, 1), none, torch.zeros(1, dtype=torch.int32, device="cuda"), none.view(0, 1), none)
    assert after.shape == (0,)
