"""Batches whose problems start anywhere: C and D with rows at multiples of 16 bytes and a batch stride that is no multiple,
so that every problem but the first starts off the 16 bytes that vector accesses need."""
import numpy as np
import pytest
import torch

import gemm_zoo_b200 as gz
from gemm_zoo_b200 import api

pytestmark = pytest.mark.gpu

TORCH = {gz.DT_F16: torch.float16, gz.DT_BF16: torch.bfloat16, gz.DT_F32: torch.float32, gz.DT_S8: torch.int8, gz.DT_S32: torch.int32}


@pytest.mark.parametrize("config,m", [(gz.CFG_AUTO, 300), (gz.CFG_1CTA_N64, 130), (gz.CFG_1CTA_N256, 130), (gz.CFG_2CTA_N128, 300),
                                      (gz.CFG_2CTA_N256, 300), (gz.CFG_2CTA_M512_N256, 600), (gz.CFG_SWAP_M16, 16), (gz.CFG_SIMT, 70)])
@pytest.mark.parametrize("in_t,out_t", [(gz.DT_BF16, gz.DT_BF16), (gz.DT_F16, gz.DT_F32), (gz.DT_S8, gz.DT_S32)])
@pytest.mark.parametrize("off_c,off_d", [(0, 1), (1, 0), (3, 5)])
def test_batch_strides_of_any_size(config, m, in_t, out_t, off_c, off_d):
    n, k, batch = 520, 128, 3
    rng = np.random.default_rng([m, off_c, off_d])
    a, b = (torch.from_numpy(rng.integers(-3, 4, (batch, r, k)).astype(np.float32)).to(TORCH[in_t]) for r in (m, n))
    sc, sd = m * n + off_c, m * n + off_d
    c = torch.from_numpy(rng.integers(-8, 9, (batch, sc)).astype(np.float32)).to(TORCH[out_t])
    for beta in (0, -2):
        d = torch.full((batch, sd), 55, dtype=TORCH[out_t], device="cuda")
        p = gz.Plan(gz.GemmDesc.make(in_t, out_t, m, n, k, gz.ROW_MAJOR, gz.COL_MAJOR, config=config, batch=batch, stride_a=m * k,
                                     stride_b=n * k, stride_c=sc, stride_d=sd))
        p.run(a.cuda(), b.cuda(), c.cuda() if beta else None, d, 1, beta)
        torch.cuda.synchronize()
        assert p.device_status()[0] == api.GZ_OK
        want = a.double() @ b.double().transpose(1, 2) + beta * c[:, :m * n].double().view(batch, m, n)
        got = d.cpu()
        assert torch.equal(got[:, :m * n].view(batch, m, n), want.to(TORCH[out_t])) and bool((got[:, m * n:] == 55).all())
