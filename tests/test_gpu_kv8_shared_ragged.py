"""kv8_shared_attention of one long prompt among single tokens: a sequence of many tiles in the kernel of few rows."""
import pytest
import torch

from test_gpu_kv8_shared import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("singles,long,at,G,D,page", [(100, 1500, 40, 4, 128, 64), (30, 700, 30, 2, 64, 16), (150, 900, 0, 8, 80, 32), (20, 333, 7, 1, 256, 128)])
@pytest.mark.parametrize("prefixes", [1, 3])
def test_one_long_prompt(dev, singles, long, at, G, D, page, prefixes):
    new = [1] * at + [long] + [1] * (singles - at)
    own = [1 + (i * 37) % 400 for i in range(at)] + [long + 50] + [1 + (i * 53) % 300 for i in range(singles - at)]
    n = singles + 1
    members = [n - 2 * (n // 3), n // 3, n // 3] if prefixes == 3 else [n]
    print(f"{singles} single tokens and {long}, G={G} D={D} page={page}, members {members}", flush=True)
    b = Batch(dev, "bf16", [300, 64, 1000][:prefixes], members, new, own, 2, G, D, page)
    got, _ = b.check()
    assert torch.equal(got, b.call())
