"""Microscaled 4-bit operators (include/gemmzoo/microscale.h) against 64-bit values (tests/mx_oracle.py).

Quantisation and its inverse are compared bit by bit.  Products: with u the half step of the output
type (2^-9 bf16 relative to the power of two above, i.e. eps / 2; fp32 2^-24) and S = sum |a||b| |alpha|,
    |D - R| <= u |R| + (K / 64 + 4) * 2^-22 * S
because the products of 4-bit values and their scales are exact, each instruction (64 elements of K)
adds its sum to the fp32 accumulator with an error of at most two units of its last place, relative to
at most S, and the epilogue rounds a handful of times.  Integer data is compared bit by bit."""
import ctypes as C
import re

import numpy as np
import pytest
import torch

import gemm_zoo_b200 as gz
from gemm_zoo_b200 import api, microscale as ms
from tests import mx_oracle as orc

FP4, NV = gz.MX_FP4, gz.MX_NVFP4
FORMATS = [FP4, NV]
HALF = {torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2, torch.float16: torch.finfo(torch.float16).eps / 2,
        torch.float32: torch.finfo(torch.float32).eps / 2}


# ------------------------------------------------------------------------------------------- CPU
def test_header_and_binding_declare_the_same_symbols():
    text = (api.PKG.parent / "include" / "gemmzoo" / "microscale.h").read_text()
    declared = set(re.findall(r"GZ_API\s+[\w ]+?\s\**(gz_\w+)\(", text))
    assert declared == set(ms.EXPORTED_SYMBOLS)
    for name in declared:
        getattr(gz.lib(), name)


def test_sizes():
    assert ms.code_pitch(1) == 16 and ms.code_pitch(32) == 16 and ms.code_pitch(33) == 32 and ms.code_pitch(4096) == 2048
    assert ms.scale_bytes(FP4, 1, 1) == 512 and ms.scale_bytes(FP4, 129, 129) == 4 * 512
    assert ms.scale_bytes(NV, 128, 64) == 512 and ms.scale_bytes(NV, 128, 65) == 1024
    assert ms.code_pitch(0) == -1 and ms.scale_bytes(3, 1, 1) == -1 and ms.scale_bytes(FP4, 0, 5) == -1
    assert ms.scale_bytes(NV, 2 ** 31 - 1024, 2 ** 31 - 1024) > 2 ** 55


@pytest.mark.parametrize("kw,expect", [
    (dict(), api.GZ_OK),
    (dict(m=0), api.GZ_ERR_INVALID_ARG), (dict(n=-1), api.GZ_ERR_INVALID_ARG), (dict(k=0), api.GZ_ERR_INVALID_ARG),
    (dict(format=3), api.GZ_ERR_INVALID_ARG), (dict(out_type=99), api.GZ_ERR_INVALID_ARG),
    (dict(out_type=gz.DT_S8), api.GZ_ERR_UNSUPPORTED), (dict(out_type=FP4), api.GZ_ERR_UNSUPPORTED),
    (dict(out_type=FP4, gated=True), api.GZ_OK), (dict(out_type=NV, gated=True), api.GZ_OK),
    (dict(config=8), api.GZ_ERR_INVALID_ARG), (dict(config=gz.MX_CFG_PAIR_N128, gated=True), api.GZ_ERR_UNSUPPORTED), (dict(split=3), api.GZ_ERR_INVALID_ARG),
    (dict(config=gz.MX_CFG_PAIR, split=8), api.GZ_ERR_UNSUPPORTED), (dict(config=gz.MX_CFG_SINGLE_N128, k=4096, split=8), api.GZ_ERR_UNSUPPORTED), (dict(config=gz.MX_CFG_SINGLE, split=8, gated=True), api.GZ_ERR_UNSUPPORTED),
    (dict(config=gz.MX_CFG_SWAP_M16, m=17), api.GZ_ERR_UNSUPPORTED),
    (dict(config=gz.MX_CFG_SWAP_M16, m=4, n=128, split=8), api.GZ_ERR_UNSUPPORTED),   # one K block
    (dict(flags=1), api.GZ_ERR_INVALID_ARG),
    (dict(pitch_a=8), api.GZ_ERR_INVALID_ARG), (dict(pitch_a=136), api.GZ_ERR_MISALIGNED),
    (dict(ldd=100), api.GZ_ERR_INVALID_ARG), (dict(ldc=255), api.GZ_ERR_INVALID_ARG),
    (dict(gated=True, out_type=NV, ldd=136), api.GZ_ERR_MISALIGNED),
    (dict(m=2 ** 31), api.GZ_ERR_TOO_LARGE), (dict(k=2 ** 40), api.GZ_ERR_TOO_LARGE),
    (dict(m=2 ** 30, n=2 ** 30), api.GZ_ERR_TOO_LARGE), (dict(m=2 ** 30, ldd=2 ** 40), api.GZ_ERR_TOO_LARGE),
    (dict(device=-1), api.GZ_ERR_INVALID_ARG),
])
def test_descriptor_checks(kw, expect):
    base = dict(format=FP4, out_type=gz.DT_BF16, m=256, n=256, k=256)
    base.update(kw)
    assert gz.mx_validate(gz.MxDesc.make(**base))[0] == expect


def test_struct_size_and_null_arguments():
    L = ms._bind()
    d = gz.MxDesc.make(FP4, gz.DT_BF16, 16, 16, 16)
    d.struct_size = 8
    assert gz.mx_validate(d)[0] == api.GZ_ERR_INVALID_ARG
    assert L.gz_mx_plan_create(None, None) == api.GZ_ERR_INVALID_ARG
    assert L.gz_mx_plan_destroy(None) == api.GZ_ERR_INVALID_ARG
    assert L.gz_mx_plan_info_get(None, None) == api.GZ_ERR_INVALID_ARG
    assert L.gz_mx_gemm_run(None, *([None] * 10)) == api.GZ_ERR_INVALID_ARG
    assert L.gz_mx_gated_run(None, *([None] * 10), 0, 1.0, None) == api.GZ_ERR_INVALID_ARG
    assert L.gz_mx_last_device_status(None, None, None) == api.GZ_ERR_INVALID_ARG


@pytest.mark.parametrize("kw,expect", [
    (dict(src=0), api.GZ_ERR_INVALID_ARG), (dict(codes=0), api.GZ_ERR_INVALID_ARG), (dict(scales=0), api.GZ_ERR_INVALID_ARG),
    (dict(rows=0), api.GZ_ERR_INVALID_ARG), (dict(k=-4), api.GZ_ERR_INVALID_ARG), (dict(format=5), api.GZ_ERR_INVALID_ARG),
    (dict(layout=2), api.GZ_ERR_INVALID_ARG), (dict(type=77), api.GZ_ERR_INVALID_ARG),
    (dict(type=gz.DT_S8), api.GZ_ERR_UNSUPPORTED), (dict(ld=63), api.GZ_ERR_INVALID_ARG),
    (dict(layout=gz.COL_MAJOR, ld=9), api.GZ_ERR_INVALID_ARG), (dict(pitch=16), api.GZ_ERR_INVALID_ARG),
    (dict(pitch=40), api.GZ_ERR_INVALID_ARG), (dict(multiplier=0.0), api.GZ_ERR_INVALID_ARG),
    (dict(multiplier=float("nan")), api.GZ_ERR_INVALID_ARG), (dict(multiplier=float("inf")), api.GZ_ERR_INVALID_ARG),
    (dict(device=-1), api.GZ_ERR_INVALID_ARG), (dict(src=4097), api.GZ_ERR_MISALIGNED),
    (dict(codes=4104), api.GZ_ERR_MISALIGNED), (dict(scales=4104), api.GZ_ERR_MISALIGNED),
    (dict(rows=2 ** 31), api.GZ_ERR_TOO_LARGE), (dict(rows=2 ** 30, k=2 ** 30, ld=2 ** 31), api.GZ_ERR_TOO_LARGE),
    (dict(rows=2 ** 30, ld=2 ** 60), api.GZ_ERR_TOO_LARGE),
])
def test_quantize_checks(kw, expect):
    """Every refusal comes before the device is touched (the addresses are never used)."""
    a = dict(src=4096, type=gz.DT_BF16, layout=gz.ROW_MAJOR, ld=0, rows=10, k=64, format=FP4, multiplier=1.0, codes=8192,
             pitch=0, scales=12288, device=0)
    a.update(kw)
    L = ms._bind()
    assert L.gz_mx_quantize(a["src"] or None, a["type"], a["layout"], a["ld"], a["rows"], a["k"], a["format"], a["multiplier"],
                            a["codes"] or None, a["pitch"], a["scales"] or None, a["device"], None) == expect
    assert L.gz_mx_dequantize(a["codes"] or None, a["pitch"], a["scales"] or None, a["format"], a["rows"], a["k"],
                              a["multiplier"], a["src"] or None, a["type"], a["layout"], a["ld"], a["device"], None) == expect


def test_without_a_gpu_there_is_no_fallback():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(gz.GzError) as e:
        gz.MxGemm(16, 16, 16, FP4, gz.DT_BF16)
    assert e.value.status == api.GZ_ERR_NO_DEVICE
    assert ms._bind().gz_mx_quantize(4096, gz.DT_BF16, 0, 0, 1, 32, FP4, 1.0, 8192, 0, 12288, 0, None) == api.GZ_ERR_NO_DEVICE


@pytest.mark.parametrize("m", [1, 16, 17, 64, 65, 128, 300, 2048, 8192])
@pytest.mark.parametrize("n", [1, 128, 4096, 14336, 100000])
@pytest.mark.parametrize("k", [1, 256, 4096, 14336])
@pytest.mark.parametrize("gated", [False, True])
def test_every_choice_can_be_launched(m, n, k, gated):
    for fmt in FORMATS:
        st, i = gz.mx_validate(gz.MxDesc.make(fmt, gz.DT_BF16, m, n, k, gated))
        assert st == api.GZ_OK and i.smem_bytes <= 232448 and i.stages >= 2
        ctas = 2 if i.config in (gz.MX_CFG_PAIR, gz.MX_CFG_PAIR_N128) else 1
        swapped = i.config in (gz.MX_CFG_SWAP_M16, gz.MX_CFG_SWAP_M32, gz.MX_CFG_SWAP_M64)
        assert i.grid >= 1 and i.grid % (ctas * i.split) == 0 and ctas * i.split <= 8 and i.split <= -(-k // 256)
        if i.split > 1 or swapped:
            assert i.grid == i.tiles * i.split * ctas
        else:
            assert i.grid <= 148


@pytest.mark.parametrize("fmt", FORMATS)
def test_scale_tiles_round_trip(fmt):
    for rows, nb in [(1, 1), (128, 4), (129, 5), (300, 9)]:
        lin = np.random.default_rng(rows).integers(0, 120, size=(rows, nb), dtype=np.uint8)
        t = gz.tile_scales(torch.from_numpy(lin), fmt)
        assert np.array_equal(t.numpy(), orc.tile(lin))
        assert np.array_equal(orc.untile(t.numpy(), rows, nb), lin)


# ------------------------------------------------------------------------------------------- GPU
gpu = pytest.mark.gpu


def _values(rows, k, dtype, seed, kind="normal"):
    rng = np.random.default_rng([seed, rows, k])
    x = rng.standard_normal((rows, k)) * np.exp2(rng.integers(-3, 4, size=(rows, 1)))
    if kind == "grid":  # quarters: many ties between codes
        x = rng.integers(-32, 33, size=(rows, k)) * 0.25
    elif kind == "wide":
        x = x * np.exp2(rng.integers(-12, 9, size=(rows, k)))
    return torch.from_numpy(x).to(dtype)


def _quantised(q):
    return (orc.unpack(q.codes.cpu().numpy()[:, :ms.code_pitch(q.k)], q.k), q.codes.cpu().numpy(), q.scales.cpu().numpy())


def _check_quantised(x64, q, fmt):
    codes, scales = orc.quantize(x64, fmt)
    got, raw, flat = _quantised(q)
    assert np.array_equal(flat[:orc.tile(scales).size], orc.tile(scales))
    assert np.array_equal(raw[:, :ms.code_pitch(q.k)], orc.pack(codes)), np.argwhere(got != codes)[:5]


SIZES = [(1, 1), (1, 4096), (2, 33), (127, 16), (128, 32), (129, 100), (64, 129), (300, 255), (5, 1000), (257, 512)]


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", [gz.ROW_MAJOR, gz.COL_MAJOR])
@pytest.mark.parametrize("kind", ["normal", "grid", "wide"])
def test_quantize_and_back_bit_for_bit(fmt, dtype, layout, kind):
    for rows, k in SIZES:
        x = _values(rows, k, dtype, 7, kind)
        xd = (x if layout == gz.ROW_MAJOR else x.t()).contiguous().cuda()
        q = gz.MxMatrix.empty(rows, k, fmt)
        q.codes.fill_(0xEE)
        q.scales.fill_(0xEE)
        gz.mx_quantize(xd, fmt, layout=layout, out=q)
        _check_quantised(x.double().numpy(), q, fmt)
        codes, scales = orc.quantize(x.double().numpy(), fmt)
        want = torch.from_numpy(orc.decode(codes, scales, fmt))
        for out in (torch.float32, dtype):
            y = torch.full(xd.shape, 77.0, dtype=out, device="cuda")
            gz.mx_dequantize(q, y, layout=layout)
            got = y.cpu() if layout == gz.ROW_MAJOR else y.cpu().t()
            assert torch.equal(got.double(), want.to(out).double())


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layout", [gz.ROW_MAJOR, gz.COL_MAJOR])
def test_quantize_strides_alignment_and_guards(fmt, layout):
    """Padded rows, an odd first element, a wider code pitch; what lies around the results stays."""
    rows, k = 70, 90
    for off, pad, dtype in [(0, 8, torch.bfloat16), (1, 3, torch.bfloat16), (3, 0, torch.float32), (16, 6, torch.float16)]:
        x = _values(rows, k, dtype, 3)
        m = x if layout == gz.ROW_MAJOR else x.t()
        flat = torch.full((off + m.shape[0] * (m.shape[1] + pad) + 8,), float("nan"), dtype=dtype, device="cuda")
        view = flat[off:off + m.shape[0] * (m.shape[1] + pad)].view(m.shape[0], -1)[:, :m.shape[1]]
        view.copy_(m)
        store = torch.full((rows, 96), 0xEE, dtype=torch.uint8, device="cuda")
        sc = torch.full((ms.scale_bytes(fmt, rows, k) + 64,), 0xEE, dtype=torch.uint8, device="cuda")
        q = gz.MxMatrix(store[:, :64], sc, rows, k, fmt)
        gz.mx_quantize(view, fmt, layout=layout, out=q)
        _check_quantised(x.double().numpy(), q, fmt)
        assert bool((store[:, ms.code_pitch(k):] == 0xEE).all()) and bool((sc[ms.scale_bytes(fmt, rows, k):] == 0xEE).all())
        back = torch.full_like(flat, 55.0)
        bview = back[off:off + m.shape[0] * (m.shape[1] + pad)].view(m.shape[0], -1)
        gz.mx_dequantize(q, bview[:, :m.shape[1]], layout=layout)
        codes, scales = orc.quantize(x.double().numpy(), fmt)
        want = torch.from_numpy(orc.decode(codes, scales, fmt))
        assert torch.equal(bview[:, :m.shape[1]].cpu().double(), (want if layout == gz.ROW_MAJOR else want.t()).to(dtype).double())
        assert bool((bview[:, m.shape[1]:] == 55.0).all()) and bool((back[:off] == 55.0).all())
        assert bool((back[off + m.shape[0] * (m.shape[1] + pad):] == 55.0).all())


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layout", [gz.ROW_MAJOR, gz.COL_MAJOR])
def test_quantize_extremes(fmt, layout):
    """Zeros, subnormals, the largest numbers, NaN and infinities: alone in a block and beside others."""
    rows, k = 12, 128
    x = np.zeros((rows, k), dtype=np.float32)
    x[1] = 1e-45
    x[2] = 3.4e38
    x[3, ::7] = -3.4e38
    x[4, 5] = np.nan
    x[5, 40] = np.inf
    x[6, 127] = -np.inf
    x[7] = np.linspace(-1e-38, 1e-38, k)
    x[8] = 2.0 ** -126
    x[9, 3] = 5e-40
    x[10] = -0.0
    x[11] = np.linspace(0, 6 * 448, k)
    t = torch.from_numpy(x)
    xd = (t if layout == gz.ROW_MAJOR else t.t()).contiguous().cuda()
    q = gz.mx_quantize(xd, fmt, layout=layout)
    _check_quantised(x.astype(np.float64), q, fmt)
    y = torch.empty_like(xd)
    gz.mx_dequantize(q, y, layout=layout)
    y = (y if layout == gz.ROW_MAJOR else y.t()).cpu().double().numpy()
    codes, scales = orc.quantize(x, fmt)
    want = orc.decode(codes, scales, fmt)
    assert np.array_equal(np.isnan(y), np.isnan(want)) and np.array_equal(y[~np.isnan(y)], want[~np.isnan(want)])
    assert np.isnan(y[4, :16]).all() and not np.isnan(y[4, 32:]).any()


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_at_every_border_of_every_scale(fmt):
    """For each scale a block of its own whose largest value gives that scale, and in it the borders between codes, the
    fp32 numbers on either side of them, and, in e4m3, largest values at and beside the borders between scales."""
    scales = orc.E4M3[1:] if fmt == NV else np.ldexp(1.0, np.arange(-100, 100))
    rows = []
    for s in scales:
        for sign in (0, 1, -1):
            b = (orc.BORDERS * s).astype(np.float32)
            assert np.array_equal(b.astype(np.float64), orc.BORDERS * s)
            b = b if sign == 0 else np.nextafter(b, np.float32(np.inf * sign), dtype=np.float32)
            top = np.float32(6 * s) if fmt == NV else np.float32(7.5 * s)
            rows.append(np.concatenate([[top], b, -b, np.zeros(1 if fmt == NV else 17, dtype=np.float32)]))
    if fmt == NV:
        mid = (orc.E4M3[1:] + orc.E4M3[:-1]) / 2 * 6
        for top in np.concatenate([np.float32(mid), np.nextafter(np.float32(mid), np.float32(0)), np.nextafter(np.float32(mid), np.float32(1e9))]):
            rows.append(np.concatenate([[top], np.linspace(0, top, 15)]))
    x = np.stack(rows).astype(np.float32)
    q = gz.mx_quantize(torch.from_numpy(x).cuda(), fmt)
    _check_quantised(x.astype(np.float64), q, fmt)


@gpu
def test_quantize_multiplier():
    x = _values(130, 200, torch.float32, 9) * 0.02
    q = gz.mx_quantize(x.cuda(), NV, multiplier=300.0)
    _check_quantised((x * 300.0).double().numpy(), q, NV)  # the product is rounded to fp32 once
    y = torch.empty(130, 200, device="cuda")
    gz.mx_dequantize(q, y, multiplier=1 / 256.0)
    codes, scales = orc.quantize((x * 300.0).double().numpy(), NV)
    assert torch.equal(y.cpu().double(), torch.from_numpy(orc.decode(codes, scales, NV) / 256.0))


def _mx(rows, k, fmt, seed, integers=False):
    """A random quantised matrix: (MxMatrix on the GPU, its values in 64 bits)."""
    rng = np.random.default_rng([seed, rows, k, fmt])
    nb = -(-k // orc.block(fmt))
    if integers:  # codes 0 +-1 +-2, scales 1 2 4
        codes = rng.choice(np.array([0, 2, 4, 10, 12], dtype=np.uint8), size=(rows, k))
        scales = rng.choice(np.array([127, 128, 129] if fmt == FP4 else [56, 64, 72], dtype=np.uint8), size=(rows, nb))
    else:
        codes = rng.integers(0, 16, size=(rows, k), dtype=np.uint8)
        scales = rng.integers(118, 131, size=(rows, nb), dtype=np.uint8) if fmt == FP4 else rng.integers(1, 90, size=(rows, nb), dtype=np.uint8)
    q = gz.MxMatrix(torch.from_numpy(orc.pack(codes)).cuda(), torch.from_numpy(orc.tile(scales)).cuda(), rows, k, fmt)
    return q, orc.decode(codes, scales, fmt)


CONFIGS = [gz.MX_CFG_PAIR, gz.MX_CFG_SINGLE, gz.MX_CFG_PAIR_N128, gz.MX_CFG_SINGLE_N128, gz.MX_CFG_SWAP_M16, gz.MX_CFG_SWAP_M32, gz.MX_CFG_SWAP_M64]
ROWS = {gz.MX_CFG_PAIR: [1, 200, 300, 520], gz.MX_CFG_SWAP_M16: [1, 13, 16], gz.MX_CFG_SWAP_M32: [1, 17, 32],
        gz.MX_CFG_SWAP_M64: [33, 64], gz.MX_CFG_SINGLE: [1, 100, 128, 257], gz.MX_CFG_PAIR_N128: [1, 300, 512],
        gz.MX_CFG_SINGLE_N128: [90, 257]}
GATED_CONFIGS = [c for c in CONFIGS if c not in (gz.MX_CFG_PAIR_N128, gz.MX_CFG_SINGLE_N128)]
GUARD = 77.0


def _out(m, n, ldd, dtype):
    full = torch.full((m + 2, ldd), GUARD, dtype=dtype, device="cuda")
    return full, full[1:m + 1]


def _guards_intact(full, m, n):
    return bool((full[0] == GUARD).all()) and bool((full[m + 1] == GUARD).all()) and bool((full[1:m + 1, n:] == GUARD).all())


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("config", CONFIGS)
def test_product_of_integers_is_exact(fmt, config):
    for m in ROWS[config]:
        for n, k in [(1, 32), (128, 256), (130, 300), (520, 1100), (400, 17)]:
            a, av = _mx(m, k, fmt, 1, True)
            b, bv = _mx(n, k, fmt, 2, True)
            full, d = _out(m, n, n + 8, torch.float32)
            plan = gz.MxGemm(m, n, k, fmt, torch.float32, ldd=n + 8, config=config, wait_limit_ns=200_000_000)
            plan(a, b, None, d[:, :n], 1.0, 0.0)
            assert plan.device_status()[0] == 0
            want = av @ bv.T
            got = d[:, :n].cpu().double().numpy()
            assert np.array_equal(got, want), (m, n, k, np.argwhere(got != want)[:6], (got != want).mean())
            assert _guards_intact(full, m, n)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("config,m,split", [(gz.MX_CFG_SWAP_M16, 5, 2), (gz.MX_CFG_SWAP_M16, 16, 4), (gz.MX_CFG_SWAP_M16, 1, 8),
                                            (gz.MX_CFG_SWAP_M32, 21, 8), (gz.MX_CFG_SWAP_M64, 50, 4), (gz.MX_CFG_SINGLE, 128, 4),
                                            (gz.MX_CFG_SINGLE, 200, 2), (gz.MX_CFG_PAIR, 300, 2),
                                            (gz.MX_CFG_PAIR, 100, 4), (gz.MX_CFG_PAIR_N128, 300, 4), (gz.MX_CFG_SINGLE_N128, 300, 4)])
def test_shared_k_ranges(fmt, config, m, split):
    for n, k in [(130, 256 * split), (256, 256 * split + 900), (300, 4096)]:
        a, av = _mx(m, k, fmt, 1, True)
        b, bv = _mx(n, k, fmt, 2, True)
        u, uv = _mx(n, k, fmt, 3, True)
        full, d = _out(m, n, n, torch.float32)
        plan = gz.MxGemm(m, n, k, fmt, torch.float32, config=config, split=split, wait_limit_ns=200_000_000)
        assert plan.info().split == split
        plan(a, b, None, d, 1.0, 0.0)
        assert plan.device_status()[0] == 0
        assert np.array_equal(d.cpu().double().numpy(), av @ bv.T) and _guards_intact(full, m, n)
        if config not in GATED_CONFIGS:
            continue
        plan = gz.MxGated(m, n, k, fmt, torch.float32, activation=gz.ACT_RELU, config=config, split=split, wait_limit_ns=200_000_000)
        plan(a, b, u, d, 2.0 ** -8, 2.0 ** -8)
        assert plan.device_status()[0] == 0
        want = (np.maximum(av @ bv.T, 0) * 2.0 ** -8).astype(np.float32) * (uv @ av.T).T.astype(np.float32) * np.float32(2.0 ** -8)
        assert np.array_equal(d.cpu().numpy(), want.astype(np.float32)) and _guards_intact(full, m, n)


def _tolerance(want, s, k, dtype):
    return HALF[dtype] * np.abs(want) + (k / 64 + 4) * 2.0 ** -22 * s + 1e-30 + (2.0 ** -25 if dtype == torch.float16 else 0)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("config,m", [(gz.MX_CFG_PAIR, 300), (gz.MX_CFG_SWAP_M16, 9), (gz.MX_CFG_SINGLE, 130), (gz.MX_CFG_PAIR_N128, 300), (gz.MX_CFG_AUTO, 70)])
def test_product_epilogue_terms(fmt, dtype, config, m):
    """alpha, beta (C apart from D and in place), bias, row and column scales; rows of D that TMA can and cannot store."""
    for n, k, ldd in [(264, 700, 264), (301, 1025, 303)]:
        rng = np.random.default_rng(m * n)
        a, av = _mx(m, k, fmt, 4)
        b, bv = _mx(n, k, fmt, 5)
        av_s, acc = np.abs(av) @ np.abs(bv).T, av @ bv.T
        alpha = float(np.float32(1.0 / acc.std()))
        c = torch.from_numpy(rng.standard_normal((m, n))).to(dtype)
        bias, rs, cs = (torch.from_numpy(rng.standard_normal(x)).float() for x in (n, m, n))
        for beta, terms, inplace in [(0.0, False, False), (-0.5, False, True), (1.0, True, False), (0.0, True, False)]:
            full, d = _out(m, n, ldd, dtype)
            if inplace:
                d[:, :n] = c.cuda()
            cc = d if inplace else torch.nn.functional.pad(c, (0, 5)).cuda()
            plan = gz.MxGemm(m, n, k, fmt, dtype, ldc=cc.stride(0), ldd=ldd, config=config, wait_limit_ns=200_000_000)
            kw = dict(bias=bias.cuda(), row_scale=rs.cuda(), col_scale=cs.cuda()) if terms else {}
            plan(a, b, cc[:, :n] if beta else None, d[:, :n], alpha, beta, **kw)
            assert plan.device_status()[0] == 0
            f = np.outer(rs.double().numpy(), cs.double().numpy()) if terms else 1.0
            want = alpha * f * acc + beta * c.double().numpy() + (bias.double().numpy() if terms else 0.0)
            s = alpha * np.abs(f) * av_s + abs(beta) * np.abs(c.double().numpy()) + (np.abs(bias.double().numpy()) if terms else 0.0)
            err = np.abs(d[:, :n].cpu().double().numpy() - want)
            assert (err <= _tolerance(want, s, k, dtype)).all(), (n, k, beta, terms, float((err / s).max()))
            assert _guards_intact(full, m, n)


ACTS = {"none": gz.ACT_NONE, "relu": gz.ACT_RELU, "gelu": gz.ACT_GELU, "gelu_tanh": gz.ACT_GELU_TANH, "silu": gz.ACT_SILU}


@gpu
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("config,m", [(gz.MX_CFG_PAIR, 260), (gz.MX_CFG_SWAP_M32, 20)])
def test_activations(act, config, m):
    """fp32 outputs.  All activations have a slope of at most 1.13, so the error of the sum grows by that; the
    approximations of exp and erf are good to 1e-6 of max(1, |x|)."""
    n, k = 200, 512
    a, av = _mx(m, k, NV, 6)
    b, bv = _mx(n, k, NV, 7)
    u, uv = _mx(n, k, NV, 8)
    acc, s = av @ bv.T, np.abs(av) @ np.abs(bv).T
    alpha = float(np.float32(1.5 / acc.std()))
    d = torch.empty(m, n, device="cuda")
    gz.MxGemm(m, n, k, NV, torch.float32, config=config)(a, b, None, d, alpha, 0.0, activation=ACTS[act])
    g = orc.act(alpha * acc, act)
    tol_g = 1.13 * (k / 64 + 4) * 2.0 ** -22 * alpha * s + 1e-6 * np.maximum(1, np.abs(alpha * acc))
    assert (np.abs(d.cpu().double().numpy() - g) <= tol_g).all()
    gz.MxGated(m, n, k, NV, torch.float32, activation=ACTS[act], config=config)(a, b, u, d, alpha, alpha)
    up, su = alpha * (av @ uv.T), alpha * (np.abs(av) @ np.abs(uv).T)
    tol = tol_g * np.abs(up) + (np.abs(g) + tol_g) * (k / 64 + 4) * 2.0 ** -22 * su + 2.0 ** -23 * np.abs(g * up)
    assert (np.abs(d.cpu().double().numpy() - g * up) <= tol).all()


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("config", GATED_CONFIGS)
def test_gated_product_shapes(fmt, config):
    """relu of integers: the gated product is exact in fp32 (|gate| and |up| below 2^12)."""
    for m in ROWS[config]:
        for n, k in [(1, 32), (128, 64), (130, 100), (300, 90), (400, 17)]:
            a, av = _mx(m, k, fmt, 1, True)
            g, gv = _mx(n, k, fmt, 2, True)
            u, uv = _mx(n, k, fmt, 3, True)
            want = np.maximum(av @ gv.T, 0) * (av @ uv.T)
            assert np.abs(want).max() < 2 ** 24
            full, d = _out(m, n, n + 4, torch.float32)
            plan = gz.MxGated(m, n, k, fmt, torch.float32, activation=gz.ACT_RELU, ldd=n + 4, config=config, wait_limit_ns=200_000_000)
            plan(a, g, u, d[:, :n])
            assert plan.device_status()[0] == 0
            got = d[:, :n].cpu().double().numpy()
            assert np.array_equal(got, want), (m, n, k, np.argwhere(got != want)[:6])
            assert _guards_intact(full, m, n)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("out", FORMATS)
@pytest.mark.parametrize("config", GATED_CONFIGS)
def test_gated_product_quantised_output(fmt, out, config):
    """Integer data: the fp32 values are exact, so codes and scales are compared bit for bit; scale rows and blocks
    that do not exist are 0, and nothing beyond a row's codes is written."""
    for m in ROWS[config]:
        for n, k in [(1, 32), (128, 64), (130, 100), (290, 90), (161, 17)]:
            a, av = _mx(m, k, fmt, 1, True)
            g, gv = _mx(n, k, fmt, 2, True)
            u, uv = _mx(n, k, fmt, 3, True)
            want = np.maximum(av @ gv.T, 0) * (av @ uv.T)
            pitch = ms.code_pitch(n) + 16
            store = torch.full((m, pitch), 0xEE, dtype=torch.uint8, device="cuda")
            sc = torch.full((ms.scale_bytes(out, m, n) + 64,), 0xEE, dtype=torch.uint8, device="cuda")
            q = gz.MxMatrix(store, sc, m, n, out)
            plan = gz.MxGated(m, n, k, fmt, out, activation=gz.ACT_RELU, ldd=pitch, config=config, wait_limit_ns=200_000_000)
            plan(a, g, u, q, out_multiplier=2.0 ** -6)
            assert plan.device_status()[0] == 0
            _check_quantised(want * 2.0 ** -6, q, out)
            assert bool((store[:, ms.code_pitch(n):] == 0xEE).all()) and bool((sc[ms.scale_bytes(out, m, n):] == 0xEE).all())


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 40, 300])
def test_nan_stays_in_its_row_and_column(fmt, m):
    n, k = 200, 300
    a, av = _mx(m, k, fmt, 1, True)
    b, bv = _mx(n, k, fmt, 2, True)
    byte = 255 if fmt == FP4 else 127
    groups = -(-(-(-k // orc.block(fmt))) // 4)
    r, c = m - 1, 77
    a.scales[(r // 128 * groups) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4] = byte
    b.scales[(c // 128 * groups) * 512 + (c % 32) * 16 + (c % 128 // 32) * 4] = byte
    d = torch.empty(m, n, device="cuda")
    gz.MxGemm(m, n, k, fmt, torch.float32)(a, b, None, d, 1.0, 0.0)
    want = av @ bv.T
    want[r], want[:, c] = np.nan, np.nan
    assert np.array_equal(d.cpu().double().numpy(), want, equal_nan=True)


@gpu
@pytest.mark.parametrize("config,m", [(gz.MX_CFG_PAIR, 200), (gz.MX_CFG_SWAP_M16, 9)])
@pytest.mark.parametrize("out", FORMATS)
def test_nan_in_a_quantised_result_stays_in_its_blocks(config, m, out):
    n, k = 200, 64
    a, av = _mx(m, k, FP4, 1, True)
    g, gv = _mx(n, k, FP4, 2, True)
    u, uv = _mx(n, k, FP4, 3, True)
    g.scales[(77 % 32) * 16 + (77 // 32) * 4] = 255  # row 77 of the gate: column 77 of the result
    q = gz.MxMatrix.empty(m, n, out)
    gz.MxGated(m, n, k, FP4, out, activation=gz.ACT_NONE, config=config)(a, g, u, q)
    want = (av @ gv.T) * (av @ uv.T)
    want[:, 77] = np.nan
    _check_quantised(want, q, out)


@gpu
@pytest.mark.parametrize("config,m,split", [(gz.MX_CFG_PAIR, 520, 1), (gz.MX_CFG_SWAP_M16, 7, 4), (gz.MX_CFG_SINGLE_N128, 200, 1)])
def test_one_plan_on_two_streams_and_in_two_graphs(config, m, split):
    """Calls of one plan may overlap: nothing is kept between them.  Eagerly on two streams, then as two graphs that
    are replayed at the same time, with operands of their own."""
    n, k = 1000, 2048
    ops = [(_mx(m, k, NV, 10 * i + 1, True), _mx(n, k, NV, 10 * i + 2, True)) for i in range(2)]
    d = [torch.empty(m, n, device="cuda") for _ in range(2)]
    plan = gz.MxGemm(m, n, k, NV, torch.float32, config=config, split=split)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    graphs = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            for _ in range(5):
                plan(ops[i][0][0], ops[i][1][0], None, d[i], 1.0, 0.0, stream=s)
    torch.cuda.synchronize()
    want = [ops[i][0][1] @ ops[i][1][1].T for i in range(2)]
    for i in range(2):
        assert np.array_equal(d[i].cpu().double().numpy(), want[i])
        d[i].zero_()
    for i, s in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            for _ in range(5):
                plan(ops[i][0][0], ops[i][1][0], None, d[i], 1.0, 0.0, stream=torch.cuda.current_stream())
        graphs.append(g)
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert np.array_equal(d[i].cpu().double().numpy(), want[i])
    assert plan.device_status()[0] == 0


@gpu
def test_padded_pitches_of_the_operands():
    """Rows of codes further apart than packed, for every operand of every kind of tile; what lies between is never read."""
    for config, m in [(gz.MX_CFG_PAIR, 260), (gz.MX_CFG_SINGLE, 130), (gz.MX_CFG_SWAP_M32, 20)]:
        n, k = 150, 330
        mats = []
        for i, rows in enumerate((m, n, n)):
            q, v = _mx(rows, k, NV, i + 1, True)
            wide = torch.full((rows, ms.code_pitch(k) + 48), 0x77, dtype=torch.uint8, device="cuda")
            wide[:, :(k + 1) // 2] = q.codes[:, :(k + 1) // 2]
            mats.append((gz.MxMatrix(wide, q.scales, rows, k, NV), v))
        p = ms.code_pitch(k) + 48
        d = torch.empty(m, n, device="cuda")
        gz.MxGemm(m, n, k, NV, torch.float32, pitch_a=p, pitch_b=p, config=config)(mats[0][0], mats[1][0], None, d, 1.0, 0.0)
        assert np.array_equal(d.cpu().double().numpy(), mats[0][1] @ mats[1][1].T)
        gz.MxGated(m, n, k, NV, torch.float32, activation=gz.ACT_NONE, pitch_a=p, pitch_b=p, config=config)(
            mats[0][0], mats[1][0], mats[2][0], d, 2.0 ** -8, 1.0)
        want = ((mats[0][1] @ mats[1][1].T) * 2.0 ** -8).astype(np.float32) * (mats[0][1] @ mats[2][1].T).astype(np.float32)
        assert np.array_equal(d.cpu().numpy(), want)


DEBUG_CHILD = """
import sys
sys.path.insert(0, {root!r})
import gemm_zoo_b200.api as api
api.lib_path = api.debug_lib_path  # before the first lib() call: this process runs the debug build
import numpy as np
import torch
import gemm_zoo_b200 as gz
from tests import test_microscale as t
for config, m in [(gz.MX_CFG_PAIR, 300), (gz.MX_CFG_SINGLE, 130), (gz.MX_CFG_PAIR_N128, 300), (gz.MX_CFG_SWAP_M16, 13), (gz.MX_CFG_SWAP_M64, 40)]:
    for n in (203, 333):
        a, av = t._mx(m, 300, gz.MX_FP4, 1, True)
        b, bv = t._mx(n, 300, gz.MX_FP4, 2, True)
        for dtype in (torch.float32, torch.bfloat16):
            d = torch.empty(m, n, dtype=dtype, device="cuda")
            p = gz.MxGemm(m, n, 300, gz.MX_FP4, dtype, config=config)
            p(a, b, None, d, 1.0, 0.0)
            assert p.device_status()[0] == 0, p.device_status()
            assert torch.equal(d.cpu(), torch.from_numpy(av @ bv.T).to(dtype))
        if config != gz.MX_CFG_PAIR_N128:
            q = gz.MxMatrix.empty(m, n, gz.MX_NVFP4)
            p = gz.MxGated(m, n, 300, gz.MX_FP4, gz.MX_NVFP4, activation=gz.ACT_RELU, config=config)
            p(a, b, b, q, 2.0 ** -8, 2.0 ** -8)
            assert p.device_status()[0] == 0, p.device_status()
print("DEBUG OK")
"""


@gpu
def test_debug_build_refuses_no_store():
    """The checked build (every plain store of the epilogue checks its coordinates first) refuses nothing."""
    import subprocess
    import sys
    from gemm_zoo_b200 import build as b
    b.build_lib(debug=True)
    root = str(api.PKG.parent)
    r = subprocess.run([sys.executable, "-c", DEBUG_CHILD.format(root=root)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "DEBUG OK" in r.stdout, (r.stdout[-500:], r.stderr[-2000:])


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 24, 200])
def test_feed_forward_chain(fmt, m):
    """quantise x -> gated product with a quantised result -> down projection, on one side stream, eagerly and from a
    graph: the launches are ordered without host synchronisation, and a replay on new inputs gives new results."""
    n, k = 384, 256
    mult = 64.0 if fmt == NV else 1.0
    rng = np.random.default_rng(m)
    wg, wu, wd = (torch.from_numpy(rng.standard_normal(s) * 0.08).float().cuda() for s in ((n, k), (n, k), (k, n)))
    qg, qu, qd = (gz.mx_quantize(w, fmt, multiplier=mult) for w in (wg, wu, wd))
    dec = [orc.decode(orc.unpack(q.codes.cpu().numpy(), q.k), orc.untile(q.scales.cpu().numpy(), q.rows, -(-q.k // orc.block(fmt))), fmt)
           for q in (qg, qu, qd)]
    x = torch.empty(m, k, dtype=torch.bfloat16, device="cuda")
    qx, qh = gz.MxMatrix.empty(m, k, fmt), gz.MxMatrix.empty(m, n, fmt)
    y = torch.empty(m, k, device="cuda")
    gated, down = gz.MxGated(m, n, k, fmt, fmt), gz.MxGemm(m, k, n, fmt, torch.float32)

    def layer(stream):
        gz.mx_quantize(x, fmt, out=qx, stream=stream)
        gated(qx, qg, qu, qh, 1 / mult, 1 / mult, stream=stream)
        down(qh, qd, None, y, 1 / mult, 0.0, stream=stream)

    def want():
        xs = orc.decode(*orc.quantize(x.cpu().double().numpy(), fmt), fmt)
        h64 = orc.act(xs @ dec[0].T / mult, "silu") * (xs @ dec[1].T / mult)
        hq = orc.decode(orc.unpack(qh.codes.cpu().numpy(), n), orc.untile(qh.scales.cpu().numpy(), m, -(-n // orc.block(fmt))), fmt)
        # the quantised h is the rounding of values within 2^-16 of h64: all but the few at a border agree
        ref = orc.decode(*orc.quantize(h64, fmt), fmt)
        assert (hq != ref).mean() < 2e-3
        return hq @ dec[2].T / mult, np.abs(hq) @ np.abs(dec[2]).T / mult

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x.copy_(torch.from_numpy(rng.standard_normal((m, k))).to(torch.bfloat16))
        layer(s)
    s.synchronize()
    ref, bound = want()
    assert (np.abs(y.cpu().double().numpy() - ref) <= _tolerance(ref, bound, n, torch.float32)).all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        layer(torch.cuda.current_stream())
    for i in range(3):
        x.copy_(torch.from_numpy(rng.standard_normal((m, k))).to(torch.bfloat16))
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        ref, bound = want()
        assert (np.abs(y.cpu().double().numpy() - ref) <= _tolerance(ref, bound, n, torch.float32)).all()
    assert gated.device_status()[0] == 0 and down.device_status()[0] == 0


@gpu
def test_python_refusals():
    x = torch.zeros(8, 64, device="cuda")
    q = gz.mx_quantize(x, FP4)
    for bad in (torch.zeros(64, device="cuda"), torch.zeros(8, 8, 8, device="cuda"), torch.zeros(8, 1, device="cuda").expand(8, 64)):
        with pytest.raises(ValueError):
            gz.mx_quantize(bad, FP4)
    with pytest.raises(ValueError):
        gz.mx_quantize(x.cpu(), FP4)
    with pytest.raises(ValueError):
        gz.mx_quantize(x.t(), FP4)
    with pytest.raises(ValueError):
        gz.mx_quantize(x, NV, out=q)
    with pytest.raises(ValueError):
        gz.mx_dequantize(q, x[:, :32])
    with pytest.raises(ValueError):
        gz.MxMatrix(q.codes[:, :16], q.scales, 8, 64, FP4)
    with pytest.raises(ValueError):
        gz.MxMatrix(q.codes, q.scales[:100], 8, 64, FP4)
    with pytest.raises(ValueError):
        gz.MxMatrix(q.codes, q.scales.cpu(), 8, 64, FP4)
    plan = gz.MxGemm(8, 8, 64, FP4, torch.float32)
    d = torch.empty(8, 8, device="cuda")
    with pytest.raises(ValueError):
        plan(q, gz.mx_quantize(x[:4], FP4), None, d, 1.0, 0.0)
    for bad in (d.half(), d[:4], d.cpu(), torch.empty(8, 16, device="cuda")[:, :8], d.t()[:, :4]):
        with pytest.raises(ValueError):
            plan(q, q, None, bad, 1.0, 0.0)
        with pytest.raises(ValueError):
            plan(q, q, bad, d, 1.0, 1.0)
    for name in ("bias", "row_scale", "col_scale"):
        for bad in (torch.zeros(7, device="cuda"), torch.zeros(8, device="cuda").half(), torch.zeros(8), torch.zeros(16, device="cuda")[::2]):
            with pytest.raises(ValueError):
                plan(q, q, None, d, 1.0, 0.0, **{name: bad})
    with pytest.raises(gz.GzError) as e:
        plan(q, q, None, d, 1.0, 1.0)  # beta without C
    assert e.value.status == api.GZ_ERR_INVALID_ARG
    with pytest.raises(gz.GzError) as e:
        plan(q, q, None, d.data_ptr() + 1, 1.0, 0.0)
    assert e.value.status == api.GZ_ERR_MISALIGNED
    h = gz.MxGated(8, 8, 64, FP4, NV)
    for bad in (d, q, None, 3):
        with pytest.raises(ValueError):
            h(q, q, q, bad)
    with pytest.raises(ValueError):
        plan(x, q, None, d, 1.0, 0.0)
    one = C.c_float(1.0)
    L = ms._bind()
    args = (q._codes_ptr, q._scales_ptr) * 3
    assert L.gz_mx_gated_run(plan._h, *args, d.data_ptr(), None, C.byref(one), C.byref(one), 4, 1.0, None) == api.GZ_ERR_INVALID_ARG
    assert L.gz_mx_gated_run(h._h, *args, d.data_ptr(), None, C.byref(one), C.byref(one), 4, 1.0, None) == api.GZ_ERR_INVALID_ARG
    assert L.gz_mx_gemm_run(h._h, *args[:4], None, d.data_ptr(), C.byref(one), C.byref(one), None, None) == api.GZ_ERR_INVALID_ARG


@gpu
@pytest.mark.parametrize("config,m,split", [(gz.MX_CFG_PAIR, 300, 1), (gz.MX_CFG_SWAP_M16, 4, 4), (gz.MX_CFG_SINGLE, 200, 1), (gz.MX_CFG_PAIR, 300, 2)])
def test_withheld_signal_times_out_and_context_survives(config, m, split):
    n, k = 300, 2048
    a, av = _mx(m, k, FP4, 1, True)
    b, bv = _mx(n, k, FP4, 2, True)
    d = torch.zeros(m, n, device="cuda")
    plan = gz.MxGemm(m, n, k, FP4, torch.float32, config=config, split=split, flags=gz.FLAG_TEST_WITHHOLD_ACC_READY, wait_limit_ns=2_000_000)
    plan(a, b, None, d, 1.0, 0.0)
    status, detail = plan.device_status()
    assert status == api.GZ_ERR_DEVICE_TIMEOUT and detail[0] in (3, 4)
    assert plan.device_status()[0] == api.GZ_OK
    gz.MxGemm(m, n, k, FP4, torch.float32, config=config, split=split)(a, b, None, d, 1.0, 0.0)
    assert np.array_equal(d.cpu().double().numpy(), av @ bv.T)


def test_in_place_conversions_are_refused():
    L = ms._bind()
    for src, codes, scales in ((4096, 4096, 8192), (4096, 8192, 4096), (4096, 8192, 8192)):
        assert L.gz_mx_quantize(src, gz.DT_BF16, 0, 0, 4, 64, FP4, 1.0, codes, 0, scales, 0, None) == api.GZ_ERR_INVALID_ARG
        assert L.gz_mx_dequantize(codes, 0, scales, FP4, 4, 64, 1.0, src, gz.DT_BF16, 0, 0, 0, None) == api.GZ_ERR_INVALID_ARG


@gpu
def test_overlapping_rows_of_codes_and_outputs_over_inputs_are_refused():
    x = torch.randn(8, 64, device="cuda")
    q = gz.mx_quantize(x, FP4)
    for codes in (q.codes[:1].expand(8, 32), torch.zeros(160, dtype=torch.uint8, device="cuda").as_strided((8, 32), (16, 1))):
        with pytest.raises(ValueError):
            gz.MxMatrix(codes, q.scales, 8, 64, FP4)
    with pytest.raises(AttributeError):
        q.codes = q.codes.clone()
    wide = torch.zeros(8, 16, device="cuda")
    plan, mixed = gz.MxGemm(8, 8, 64, FP4, torch.float32), gz.MxGemm(8, 8, 64, FP4, torch.float32, ldc=16)
    d = wide[:, :8].contiguous()
    with pytest.raises(gz.GzError):
        plan(q, q, None, q.codes.data_ptr(), 1.0, 0.0)
    with pytest.raises(gz.GzError):
        mixed(q, q, d.data_ptr(), d, 1.0, 1.0)
    mixed(q, q, wide[:, :8], d, 1.0, 1.0)
    chain = gz.MxGated(8, 64, 64, FP4, FP4)
    out = gz.MxMatrix.empty(8, 64, FP4)
    up = gz.mx_quantize(torch.randn(64, 64, device="cuda"), FP4)
    chain(q, up, up, out)
    for bad in (q, gz.MxMatrix(out.codes, q.scales, 8, 64, FP4), gz.MxMatrix(q.codes, out.scales, 8, 64, FP4)):
        with pytest.raises(gz.GzError):
            chain(q, up, up, bad)
    torch.cuda.synchronize()


@gpu
def test_new_matrices_belong_to_the_stream_that_writes_them():
    """What mx_quantize allocates is freed in the order of the stream it was given, not of the current one."""
    x = torch.randn(256, 1024, device="cuda")
    want = gz.mx_quantize(x, NV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (side, side.cuda_stream, None, 0):
        q = gz.mx_quantize(x, NV, stream=stream)
        with torch.cuda.stream(side):
            r = gz.mx_quantize(x, NV, stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(q.codes, want.codes) and torch.equal(r.codes, want.codes) and torch.equal(r.scales, want.scales)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layout", [gz.ROW_MAJOR, gz.COL_MAJOR])
def test_quantise_and_decode_beyond_32_bit_offsets(fmt, layout):
    """2.6e9 values: the last rows come out as those rows alone do."""
    rows, k, tail = 40000, 65536, 64  # (the tail starts at a whole row group of the scales)
    shape = (rows, k) if layout == gz.ROW_MAJOR else (k, rows)
    x = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_()
    last = (x[-tail:] if layout == gz.ROW_MAJOR else x[:, -tail:]).contiguous()
    q, w = gz.mx_quantize(x, fmt, layout=layout), gz.mx_quantize(last, fmt, layout=layout)
    assert (rows - tail) % 128 == 0
    assert torch.equal(q.codes[-tail:], w.codes) and torch.equal(q.scales[-w.scales.numel():], w.scales)
    back = gz.mx_dequantize(q, x, layout=layout)
    assert torch.equal((back[-tail:] if layout == gz.ROW_MAJOR else back[:, -tail:]), gz.mx_dequantize(w, last, layout=layout))


@gpu
@pytest.mark.parametrize("config", [gz.MX_CFG_PAIR, gz.MX_CFG_SINGLE_N128])
def test_products_beyond_32_bit_offsets(config):
    """A result of 2.6e9 values, C and D: the last rows come out as those rows alone do."""
    m, n, k, tail = 40000, 65536, 64, 64
    (a, _), (b, _) = _mx(m, k, NV, 1, True), _mx(n, k, NV, 2, True)
    d = torch.ones(m, n, dtype=torch.float16, device="cuda")
    gz.MxGemm(m, n, k, NV, torch.float16, config=config)(a, b, d, d, 1.0 / 64, 2.0)
    blocks = -(-k // 64) * 512
    rest = gz.MxMatrix(a.codes[-tail:], a.scales[(m - tail) // 128 * blocks:], tail, k, NV)
    want = torch.ones(tail, n, dtype=torch.float16, device="cuda")
    gz.MxGemm(tail, n, k, NV, torch.float16)(rest, b, want, want, 1.0 / 64, 2.0)
    assert (m - tail) % 128 == 0 and torch.equal(d[-tail:], want)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("config,split", [(gz.MX_CFG_PAIR, 1), (gz.MX_CFG_SINGLE, 2), (gz.MX_CFG_PAIR_N128, 1), (gz.MX_CFG_SINGLE_N128, 4), (gz.MX_CFG_SWAP_M64, 1)])
@pytest.mark.parametrize("gated", [False, True])
def test_nothing_beside_the_result_is_written(dtype, config, split, gated):
    """Results whose rows end anywhere within 16 bytes, in a matrix whose rows start at multiples of 16 bytes."""
    if gated and config in (gz.MX_CFG_PAIR_N128, gz.MX_CFG_SINGLE_N128):
        return
    m, k, step = 60, 1100, 16 // torch.empty(0, dtype=dtype).element_size()
    (a, av) = _mx(m, k, FP4, 1, True)
    for n in (256 + step, 257, 258, 259, 385, 387):
        (b, bv), (u, uv) = _mx(n, k, FP4, n, True), _mx(n, k, FP4, n + 1000, True)
        full, d = _out(m, n, -(-n // step) * step + step, dtype)
        if gated:
            gz.MxGated(m, n, k, FP4, dtype, activation=gz.ACT_RELU, ldd=full.stride(0), config=config, split=split)(a, b, u, d[:, :n])
            want = np.maximum(av @ bv.T, 0) * (av @ uv.T)
        else:
            gz.MxGemm(m, n, k, FP4, dtype, ldd=full.stride(0), config=config, split=split)(a, b, None, d[:, :n], 1.0, 0.0)
            want = av @ bv.T
        torch.cuda.synchronize()
        assert torch.equal(d[:, :n].cpu(), torch.from_numpy(want).float().to(dtype))
        assert _guards_intact(full, m, n)
