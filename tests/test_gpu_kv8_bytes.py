"""kv8_read over every scale byte and every code, against the oracle: bit for bit where the type holds the value."""
import numpy as np
import pytest
import torch

from oracle import mx_ref as ref
from test_gpu_kv8 import DT, _i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_every_byte_and_code(dev, dtype):
    """256 pages, one for each scale byte, that hold all 256 codes.  fp32 holds every value; the 16-bit types round
    those below their normal range (bf16: half a step of 2^-133, fp16: of 2^-24) and fp16 those above it to infinity."""
    import metalops_amd as mo
    codes = np.tile(np.arange(256, dtype=np.uint8).reshape(1, 1, 16, 16), (256, 1, 1, 1))
    scales = np.arange(256, dtype=np.uint8).reshape(256, 1)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    cache = mo.KV8Cache(t(codes), t(codes.swapaxes(2, 3)), t(scales), t(scales))
    k, v = mo.kv8_read(cache, _i32(np.arange(256).reshape(256, 1), dev), _i32([16] * 256, dev), DT[dtype])
    want = (ref.e4m3_decode(codes) * ref.scale_value(scales)[..., None, None]).transpose(0, 2, 1, 3)
    exact = torch.from_numpy(want)
    for got in (k, v):
        got = got.cpu()
        assert torch.equal(got.isnan(), exact.isnan())
        if dtype == "f32":
            assert torch.equal(got.double().nan_to_num(7.0), torch.where(exact.abs() > torch.finfo(torch.float32).max, exact.sign() * float("inf"), exact).nan_to_num(7.0))
            continue
        info = torch.finfo(DT[dtype])
        small, large = exact.abs() < info.tiny, exact.abs() > info.max
        ok = ~(small | large | exact.isnan())
        assert torch.equal(got[ok].double(), exact[ok])
        assert ((got.double() - exact)[small].abs() <= info.tiny * info.eps / 2).all()
        assert (got[large].abs() >= info.max).all()
