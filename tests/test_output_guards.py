"""D as part of a wider matrix whose rows start at multiples of 16 bytes while its own rows end anywhere: what lies
behind each row stays as it was.  (A TMA store whose box ends within 16 bytes writes zeros up to the next multiple.)"""
import numpy as np
import pytest
import torch

import gemm_zoo_b200 as gz
from gemm_zoo_b200 import api
from oracle import cpu_oracle as orc
from tests.helpers import Case, check, make_operands, run_gpu

pytestmark = pytest.mark.gpu

F16, BF16, F32, S8, S32, E4M3 = gz.DT_F16, gz.DT_BF16, gz.DT_F32, gz.DT_S8, gz.DT_S32, gz.DT_E4M3
CONFIGS = [gz.CFG_1CTA_N256, gz.CFG_1CTA_N128, gz.CFG_1CTA_N64, gz.CFG_2CTA_N256, gz.CFG_2CTA_N128,
           gz.CFG_2CTA_M512_N256, gz.CFG_SWAP_M64]
PER16 = {F16: 8, BF16: 8, F32: 4, S32: 4}


def _pad(n, out_t):
    """Elements behind a row: up to the next multiple of 16 bytes, and 16 bytes more."""
    return -n % PER16[out_t] + PER16[out_t]


def _check(case):
    """tests.helpers.check; its oracle takes C as integers for s8 inputs, so a dequantising product is computed here."""
    if case.in_type != S8 or case.out_type == S32:
        return check(case)
    a, b, c = make_operands(case)
    out, guard_ok, info, (status, _) = run_gpu(case, a, b, c)
    acc = orc.gemm_s8(a.numpy(), b.numpy(), None, case.m, case.n, case.k, a_col_major=case.a_col, b_col_major=case.b_col,
                      lda=case.lda, ldb=case.ldb)
    want = orc.round_to(case.out_type, case.alpha * acc + case.beta * c[:, :case.n].double().numpy())
    return {"case": case.name(), "epilogue_tma": info.epilogue_tma, "guard_ok": guard_ok, "status": status,
            "ok": guard_ok and status == 0 and torch.equal(out, want)}


@pytest.mark.parametrize("config", CONFIGS)
@pytest.mark.parametrize("in_t,out_t", [(F16, F16), (F16, F32), (BF16, BF16), (BF16, F32), (F32, F32), (S8, S32), (S8, F16),
                                        (S8, BF16), (S8, F32), (E4M3, F16), (E4M3, BF16), (E4M3, F32)])
def test_every_output_type_and_tile(config, in_t, out_t):
    m = 60 if config == gz.CFG_SWAP_M64 else 300
    for n in (1, 63, 129, 517, 518, 519, 765):
        for beta, flags in ((0, 0), (-2, 0), (0, gz.FLAG_EPILOGUE_TMA)):
            r = _check(Case(in_t, out_t, m, n, 128, b_col=True, config=config, alpha=1, beta=beta, flags=flags, pad_d=_pad(n, out_t)))
            assert r["ok"], r
            assert config == gz.CFG_SWAP_M64 or r["epilogue_tma"] == 1


@pytest.mark.parametrize("out_t", [BF16, F32])
def test_many_tiles_and_the_chosen_configuration(out_t):
    """Tail strips, the 512x256 tile with and without C, D in place of C."""
    for m, n, config in ((2304, 2051, gz.CFG_AUTO), (2304, 2051, gz.CFG_2CTA_N256), (4096, 3001, gz.CFG_2CTA_M512_N256), (1, 4099, gz.CFG_AUTO)):
        for beta, inplace in ((0, False), (1, True)):
            r = check(Case(BF16, out_t, m, n, 64, b_col=True, config=config, alpha=1, beta=beta, inplace=inplace, pad_d=_pad(n, out_t)))
            assert r["ok"], r


@pytest.mark.parametrize("out_t", [F16, F32])
@pytest.mark.parametrize("config", [gz.CFG_AUTO, gz.CFG_2CTA_N256, gz.CFG_1CTA_N64])
def test_batches(out_t, config):
    m, n, k, batch = 130, 261, 64, 3
    ldd = n + _pad(n, out_t)
    dtype = torch.float16 if out_t == F16 else torch.float32
    rng = np.random.default_rng(1)
    a, b = (torch.from_numpy(rng.integers(-3, 4, (batch, r, k)).astype(np.float32)).half().cuda() for r in (m, n))
    d = torch.full((batch, m + 1, ldd), 77.0, dtype=dtype, device="cuda")
    g = gz.Plan(gz.GemmDesc.make(F16, out_t, m, n, k, gz.ROW_MAJOR, gz.COL_MAJOR, ldd=ldd, config=config, batch=batch,
                                 stride_a=m * k, stride_b=n * k, stride_c=m * n, stride_d=(m + 1) * ldd))
    assert g.info().epilogue_tma == 1
    g.run(a, b, None, d, 1.0, 0.0)
    torch.cuda.synchronize()
    assert g.device_status()[0] == api.GZ_OK
    want = a.double().cpu() @ b.double().cpu().transpose(1, 2)
    got = d.cpu()
    assert torch.equal(got[:, :m, :n].double(), want)
    assert bool((got[:, :m, n:] == 77).all()) and bool((got[:, m] == 77).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("config", [gz.CFG_1CTA_N128, gz.CFG_2CTA_N256, gz.CFG_2CTA_M512_N256])
def test_epilogue_terms(dtype, config):
    m, n, k = 300, 523, 64
    out_t = BF16 if dtype == torch.bfloat16 else F32
    ldd = n + _pad(n, out_t)
    rng = np.random.default_rng(2)
    a, b = (torch.from_numpy(rng.integers(-3, 4, (r, k)).astype(np.float32)).bfloat16().cuda() for r in (m, n))
    bias = torch.from_numpy(rng.integers(-9, 10, n).astype(np.float32))
    d = torch.full((m, ldd), 77.0, dtype=dtype, device="cuda")
    g = gz.Plan(gz.GemmDesc.make(BF16, out_t, m, n, k, gz.ROW_MAJOR, gz.COL_MAJOR, ldd=ldd, config=config))
    g.run_ex(a, b, None, d, 1.0, 0.0, bias=bias.cuda(), activation=gz.ACT_RELU)
    torch.cuda.synchronize()
    assert g.device_status()[0] == api.GZ_OK
    want = torch.relu(a.double().cpu() @ b.double().cpu().t() + bias.double())
    assert torch.equal(d[:, :n].cpu(), want.to(dtype)) and bool((d[:, n:] == 77).all())
