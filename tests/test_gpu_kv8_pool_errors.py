"""An error that an earlier HIP call has left: the pool's calls report it and change nothing."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

I32 = torch.int32


def _hip():
    with open("/proc/self/maps") as f:
        return ctypes.CDLL(next(line.split()[-1] for line in f if "libamdhip64" in line))


@pytest.mark.parametrize("native", [True, False])
def test_counts_change_once(dev, native, monkeypatch):
    import metalops_amd as mo
    from metalops_amd import pool as module
    if not native:
        monkeypatch.setattr(module, "_native", None)
    hip = _hip()
    pool = mo.KV8Pool.empty(2, 12, 1, 16, 16, dev)
    ints = lambda x: torch.tensor(x, dtype=I32, device=dev)
    table, lens = pool.table(2, 3), ints([20, 5])
    assert mo.kv8_resize(pool, table, ints([0, 0]), lens).item() == 0
    args = {k: ints(v) for k, v in dict(three=[0, 0, 1], two=[0, 1], more=[40, 17], fewer=[0, 1], src=[0], dst=[9]).items()}
    calls = {
        "fork": lambda: mo.kv8_fork(pool, table, lens, args["three"]),
        "release": lambda: mo.kv8_fork(pool, table, lens, args["two"], release=True),
        "grow": lambda: mo.kv8_resize(pool, table, lens, args["more"]),
        "shrink": lambda: mo.kv8_resize(pool, table, lens, args["fewer"]),
        "compact": lambda: mo.kv8_compact(pool, table),
        "copy": lambda: mo.kv8_copy_pages(pool, args["src"], args["dst"]),
    }
    for name, call in calls.items():
        refs, rows = pool.refs.clone(), table.clone()
        torch.cuda.synchronize()
        hip.hipGetLastError()
        assert hip.hipSetDevice(1 << 20) != 0        # refused by the runtime, which keeps the error
        with pytest.raises(RuntimeError, match="earlier call" if native else None):      # torch's own calls may be the first to see it
            call()
        torch.cuda.synchronize()
        assert torch.equal(pool.refs, refs) and torch.equal(table, rows), name
        assert hip.hipGetLastError() == 0
    rows, n = mo.kv8_fork(pool, table, lens, ints([0, 0, 1]))
    assert pool.refs.sum().item() == 3 + 5
