"""Plans whose bins are counted by another lane of a wave in every turn of 64 tokens."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 3, 64, 4096])
@pytest.mark.parametrize("turns", [2, 9, 33, 300])
def test_a_bin_counted_by_other_lanes_in_turn(gpu, n, turns):
    from looped_blockell import kernels as K
    print(f"plan of {turns} turns, {n} adapters", flush=True)
    lane, t = torch.arange(64)[None, :], torch.arange(turns)[:, None]
    for step in (1, 5, 63):
        first = (t * step) % 64                         # the first lane that holds bin 0 in this turn
        ids = torch.where(lane >= first, torch.zeros_like(lane + t), torch.full_like(lane + t, n - 1))
        ids[(lane + t) % 7 == 0] = -1
        ids = ids.flatten()[:64 * turns - 13]
        plan = K.adapter_plan(ids.to(torch.int32).to(gpu), n)
        bins = torch.where(ids < 0, torch.full_like(ids, n), ids)
        count = torch.bincount(bins, minlength=n + 1)
        data = plan.data.cpu().long()
        assert torch.equal(data[:n + 2], torch.cat([torch.zeros(1, dtype=torch.long), count.cumsum(0)]))
        N, w = len(ids), (n + 3) // 2 * 2
        at = 2 * w + 4 * (N // 64 + min(N, n + 1))
        assert torch.equal(data[at:at + N], torch.argsort(bins, stable=True))
