"""Calls of the microscaled operators that tests/test_microscale.py does not make."""
import ctypes as C

import numpy as np
import pytest
import torch

import gemm_zoo_b200 as gz
from gemm_zoo_b200 import api, microscale as ms
from tests import mx_oracle as orc
from tests.test_microscale import (ACTS, FORMATS, FP4, HALF, NV, _check_quantised, _guards_intact, _mx, _out, _tolerance,
                                   _values)

gpu = pytest.mark.gpu


# ------------------------------------------------------------------------------------------- shuffles
def test_shuffle_masks_do_not_depend_on_convergence():
    """Which lanes happen to be together (__activemask) says nothing about which lanes share a scale word."""
    for f in (api.PKG / "csrc").rglob("*.cu*"):
        assert "__activemask" not in f.read_text(), f


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_whose_words_end_inside_a_warp(fmt, dtype):
    """Every number of scale words of a row up to a whole block of threads, and rows in several pieces."""
    word = 64 if fmt == NV else 128
    for words in [1, 2, 3, 5, 6, 7, 9, 11, 13, 21, 31, 32, 33, 43, 63, 65]:
        for k in (words * word, words * word - 17):
            x = _values(5, k, dtype, 11)
            _check_quantised(x.double().numpy(), gz.mx_quantize(x.cuda(), fmt), fmt)


# ------------------------------------------------------------------------------------------- shared K ranges
@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("out", FORMATS)
@pytest.mark.parametrize("config,m,split", [(gz.MX_CFG_SWAP_M16, 1, 2), (gz.MX_CFG_SWAP_M16, 13, 4), (gz.MX_CFG_SWAP_M16, 16, 8),
                                            (gz.MX_CFG_SWAP_M32, 21, 8), (gz.MX_CFG_SWAP_M32, 32, 2), (gz.MX_CFG_SWAP_M64, 50, 4),
                                            (gz.MX_CFG_SWAP_M64, 64, 8), (gz.MX_CFG_SINGLE, 100, 2), (gz.MX_CFG_SINGLE, 130, 4),
                                            (gz.MX_CFG_PAIR, 100, 2), (gz.MX_CFG_PAIR, 300, 2), (gz.MX_CFG_PAIR, 200, 4)])
def test_quantised_gated_result_with_a_shared_k_range(fmt, out, config, m, split):
    """Integer sums: codes and scales bit for bit, scale rows and blocks that do not exist 0, nothing else written."""
    for n, k in [(1, 256 * split), (130, 256 * split + 17), (290, 256 * split + 900), (200, 4096)]:
        (a, av), (g, gv), (u, uv) = _mx(m, k, fmt, 1, True), _mx(n, k, fmt, 2, True), _mx(n, k, fmt, 3, True)
        sums = av @ gv.T, av @ uv.T
        assert all(np.abs(s).max() < 2 ** 24 for s in sums)
        # two roundings to fp32 at most: none of the scaled sums (powers of two), one of their product
        want = (np.maximum(sums[0], 0) * 2.0 ** -8).astype(np.float32) * (sums[1] * 2.0 ** -8).astype(np.float32)
        pitch, size = ms.code_pitch(n) + 16, ms.scale_bytes(out, m, n)
        store = torch.full((m + 1, pitch), 0xEE, dtype=torch.uint8, device="cuda")
        sc = torch.full((size + 64,), 0xEE, dtype=torch.uint8, device="cuda")
        q = gz.MxMatrix(store[:m], sc, m, n, out)
        plan = gz.MxGated(m, n, k, fmt, out, activation=gz.ACT_RELU, ldd=pitch, config=config, split=split, wait_limit_ns=200_000_000)
        assert plan.info().split == split
        plan(a, g, u, q, 2.0 ** -8, 2.0 ** -8, 2.0 ** -3)
        assert plan.device_status()[0] == 0
        _check_quantised(want.astype(np.float64) * 2.0 ** -3, q, out)
        assert bool((store[:m, ms.code_pitch(n):] == 0xEE).all()) and bool((store[m] == 0xEE).all()) and bool((sc[size:] == 0xEE).all())


SHARED = [(gz.MX_CFG_PAIR, 300, 2), (gz.MX_CFG_PAIR, 100, 4), (gz.MX_CFG_SINGLE, 200, 2), (gz.MX_CFG_SINGLE, 130, 8),
          (gz.MX_CFG_PAIR_N128, 300, 2), (gz.MX_CFG_PAIR_N128, 520, 4), (gz.MX_CFG_SINGLE_N128, 130, 2), (gz.MX_CFG_SINGLE_N128, 100, 4),
          (gz.MX_CFG_SWAP_M16, 9, 8), (gz.MX_CFG_SWAP_M32, 20, 2), (gz.MX_CFG_SWAP_M64, 64, 4)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("config,m,split", SHARED)
def test_epilogue_terms_with_a_shared_k_range(dtype, config, m, split):
    """C apart from D and in place, rows of C and D aligned and not, bias, row and column scales, ReLU.  Integers and powers
    of two: every fp32 value is exact, so results are compared bit for bit after the one rounding to the output type."""
    step = 16 // torch.empty(0, dtype=dtype).element_size()
    for n, k, odd in [(264, 256 * split, 0), (261, 256 * split + 800, 3), (520, 256 * split + 15, step)]:
        rng = np.random.default_rng([m, n, split])
        (a, av), (b, bv) = _mx(m, k, NV, 4, True), _mx(n, k, NV, 5, True)
        acc = av @ bv.T
        c = rng.integers(-64, 65, (m, n)).astype(np.float64)
        bias = rng.integers(-64, 65, n).astype(np.float32)
        rs, cs = (2.0 ** rng.integers(-3, 2, r).astype(np.float32) for r in (m, n))
        ldd = -(-n // step) * step + odd
        for beta, terms, inplace in [(0.0, True, False), (-2.0, False, True), (-2.0, False, False), (3.0, True, True), (3.0, True, False)]:
            full, d = _out(m, n, ldd, dtype)
            cd = torch.from_numpy(c).to(dtype)
            if inplace:
                d[:, :n] = cd.cuda()
                cc = d
            else:
                cc = torch.nn.functional.pad(cd, (0, odd)).cuda()
            plan = gz.MxGemm(m, n, k, NV, dtype, ldc=cc.stride(0), ldd=ldd, config=config, split=split, wait_limit_ns=200_000_000)
            assert plan.info().split == split
            kw = dict(bias=torch.from_numpy(bias).cuda(), row_scale=torch.from_numpy(rs).cuda(), col_scale=torch.from_numpy(cs).cuda(),
                      activation=gz.ACT_RELU) if terms else {}
            plan(a, b, cc[:, :n] if beta else None, d[:, :n], 0.5, beta, **kw)
            assert plan.device_status()[0] == 0
            want = 0.5 * acc * (np.outer(rs.astype(np.float64), cs) if terms else 1.0) + beta * c + (bias if terms else 0.0)
            assert np.abs(want).max() * 2.0 ** 6 < 2 ** 24  # in units of 2^-6, what the scales divide by
            if terms:
                want = np.maximum(want, 0)
            assert torch.equal(d[:, :n].cpu(), torch.from_numpy(want).float().to(dtype)), (n, k, beta, terms, inplace)
            assert _guards_intact(full, m, n)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", [(1, 1024, 4096), (64, 512, 4096), (200, 512, 8192)])
def test_chosen_configurations_share_the_k_range(fmt, m, n, k):
    """The sizes of decoding steps, with the tile and split that are chosen for them; quantised and plain results."""
    (a, av), (g, gv), (u, uv) = _mx(m, k, fmt, 1, True), _mx(n, k, fmt, 2, True), _mx(n, k, fmt, 3, True)
    sums = av @ gv.T, av @ uv.T
    assert all(np.abs(s).max() < 2 ** 24 for s in sums)
    want = (np.maximum(sums[0], 0) * 2.0 ** -8).astype(np.float32) * (sums[1] * 2.0 ** -8).astype(np.float32)
    for out in (fmt, torch.float32):
        plan = gz.MxGated(m, n, k, fmt, out, activation=gz.ACT_RELU)
        assert plan.info().split > 1
        d = gz.MxMatrix.empty(m, n, out) if out is fmt else torch.empty(m, n, device="cuda")
        plan(a, g, u, d, 2.0 ** -8, 2.0 ** -8)
        if out is fmt:
            _check_quantised(want.astype(np.float64), d, fmt)
        else:
            assert np.array_equal(d.cpu().numpy(), want)
    d = torch.empty(m, n, device="cuda")
    plan = gz.MxGemm(m, n, k, fmt, torch.float32)
    plan(a, g, None, d, 1.0, 0.0)
    assert plan.info().split > 1 and np.array_equal(d.cpu().double().numpy(), sums[0])


# ------------------------------------------------------------------------------------------- aliases
@gpu
@pytest.mark.parametrize("config", [gz.MX_CFG_SWAP_M16, gz.MX_CFG_SINGLE_N128, gz.MX_CFG_PAIR])
def test_a_result_in_place_of_an_epilogue_vector_is_refused(config):
    a, b = gz.mx_quantize(torch.randn(1, 256, device="cuda"), NV), gz.mx_quantize(torch.randn(300, 256, device="cuda"), NV)
    plan, d = gz.MxGemm(1, 300, 256, NV, torch.float32, config=config), torch.ones(1, 300, device="cuda")
    for name, v in (("bias", d[0]), ("col_scale", d[0]), ("row_scale", d[0, :1])):
        with pytest.raises(gz.GzError) as e:
            plan(a, b, None, d, 1.0, 0.0, **{name: v})
        assert e.value.status == api.GZ_ERR_INVALID_ARG
    torch.cuda.synchronize()
    assert bool((d == 1).all())
    plan(a, b, None, d, 1.0, 0.0, bias=torch.zeros(300, device="cuda"))
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------- decoding
@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layout", [gz.ROW_MAJOR, gz.COL_MAJOR])
@pytest.mark.parametrize("multiplier", [1.0, -1.0, 2.0 ** -10, 0.3, -0.9999999, 1.7, 2.0 ** -140, -3e38, 1e-38])
def test_every_code_of_every_scale_decodes_to_its_product(fmt, layout, multiplier):
    """code * scale * multiplier, rounded once to fp32 and once to the type, to infinity only where the product is beyond it."""
    size, count = orc.block(fmt), 256 if fmt == FP4 else 128
    codes = np.tile(np.arange(16, dtype=np.uint8), (count, size // 16))
    scales = np.arange(count, dtype=np.uint8)[:, None]
    q = gz.MxMatrix(torch.from_numpy(orc.pack(codes)).cuda(), torch.from_numpy(orc.tile(scales)).cuda(), count, size, fmt)
    with np.errstate(over="ignore", invalid="ignore"):
        want = (orc.decode(codes, scales, fmt) * float(np.float32(multiplier))).astype(np.float32)  # 2 + 24 bits: exact in 64
    for dtype in (torch.float32, torch.bfloat16):
        y = torch.empty((count, size) if layout == gz.ROW_MAJOR else (size, count), dtype=dtype, device="cuda")
        gz.mx_dequantize(q, y, layout=layout, multiplier=multiplier)
        got = y.cpu() if layout == gz.ROW_MAJOR else y.cpu().t()
        ref = torch.from_numpy(want).to(dtype)
        assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(got[~torch.isnan(got)], ref[~torch.isnan(ref)])


# ------------------------------------------------------------------------------------------- activations
def _activated(x, act, config, m):
    """act of the values x: the bias of a product that is zero."""
    n = x.numel()
    a, b = gz.mx_quantize(torch.zeros(m, 64, device="cuda"), FP4), gz.mx_quantize(torch.zeros(n, 64, device="cuda"), FP4)
    d = torch.empty(m, n, device="cuda")
    gz.MxGemm(m, n, 64, FP4, torch.float32, config=config)(a, b, None, d, 1.0, 0.0, bias=x.cuda(), activation=ACTS[act])
    d = d.cpu()
    assert all(torch.equal(d[i], d[0]) for i in range(m)) or bool(torch.isnan(x).any())
    return d[0].double().numpy()


@gpu
@pytest.mark.parametrize("config,m", [(gz.MX_CFG_SWAP_M16, 2), (gz.MX_CFG_PAIR, 130)])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_activations_over_their_range(act, config, m):
    """The absolute bound (5e-7 |x|) and the relative one where the result is small.

    With u = 2^-24 and __expf good to (2 + 1.173 |y|) * 2u: e^y is off by at most |y| * (y's own relative error, 6u for
    the tanh form's argument, 0 for SiLU's, 1.173 * 2u for __expf) + 4u, relative; a sigmoid s = 1 / (1 + e^y) by (1 - s)
    times that, + 4u for the sum, the approximate reciprocal and the product: 5e-7 |y| + 6e-7 relative, and, as
    s (1 - s) |y| < 0.23 and s (1 - s) <= 1/4, 4e-7 absolute.  erfc(z) = p(t) t e^(-z^2) is good to 1.5e-7 by its
    source; its factors' roundings are at most 5u + 7u z^2 (e^(-z^2) z^2 < 0.37) and __expf's, below 1e-6 together, and
    x / 2 times it is off by half of both; against that formula in 64 bits it is within 1.5e-6 + 5e-7 z^2, relative."""
    x = torch.cat([torch.linspace(-9, 9, 40001), torch.randn(4000) * 1e-3, torch.randn(4000) * 40, torch.randn(500) * 1e-30])
    got, xd = _activated(x, act, config, m), x.double().numpy()
    erfc = np.vectorize(__import__("math").erfc)
    if act == "gelu":
        want = 0.5 * xd * erfc(-xd / np.sqrt(2))
    else:
        y = -xd if act == "silu" else -2 * np.sqrt(2 / np.pi) * (xd + 0.044715 * xd ** 3)
        with np.errstate(over="ignore"):
            want = xd / (1 + np.exp(y))
        normal = y < 80
        assert (np.abs(got - want)[normal] <= ((6e-7 + 5e-7 * np.abs(y)) * np.abs(want) + 2.0 ** -126)[normal]).all()
    assert (np.abs(got - want) <= 5e-7 * np.abs(xd) + 2.0 ** -126).all()
    if act == "gelu":
        z = np.abs(xd) / np.sqrt(2)
        t = 1 / (1 + 0.3275911 * z)
        c = t * (0.254829592 + t * (-0.284496736 + t * (1.421413741 + t * (-1.453152027 + t * 1.061405429)))) * np.exp(-z * z)
        form = 0.5 * xd * c
        some = (xd < 0) & (z < 8)
        assert (np.abs(got - form)[some] <= ((1.5e-6 + 5e-7 * z * z) * np.abs(form) + 2.0 ** -126)[some]).all()
        for low, bound in ((-3, 1e-4), (-4.5, 1e-3), (-7.5, 1e-2)):
            assert (np.abs(got - want)[xd >= low] <= bound * np.abs(want)[xd >= low] + 2.0 ** -126).all()


@gpu
@pytest.mark.parametrize("config,m", [(gz.MX_CFG_SWAP_M16, 2), (gz.MX_CFG_PAIR, 130)])
@pytest.mark.parametrize("act", list(ACTS))
def test_activations_of_infinities_and_large_numbers(act, config, m):
    big = torch.tensor([float("inf"), 3e38, 1e20, -1e20, -3e38, 0.0, float("nan"), float("-inf")])
    got = _activated(big, act, config, m)
    assert np.array_equal(got[:3], big[:3].double().numpy())
    if act == "none":
        assert np.array_equal(got[3:], big[3:].double().numpy(), equal_nan=True)
    else:
        assert (got[3:6] == 0).all() and np.isnan(got[6])
        # the formulas give -inf * 0 except for relu
        assert got[7] == 0 if act == "relu" else np.isnan(got[7])


@gpu
@pytest.mark.parametrize("act", list(ACTS))
def test_gated_product_of_large_gates(act):
    """A gate far from zero: act(gate) is gate or 0, and times up exactly that."""
    m, n, k = 17, 96, 64
    a = gz.mx_quantize(torch.ones(m, k, device="cuda"), FP4)
    sign = torch.where(torch.arange(n) % 2 == 0, 1.0, -1.0)[:, None].expand(n, k).contiguous().cuda()
    g, u = gz.mx_quantize(sign, FP4), gz.mx_quantize(torch.ones(n, k, device="cuda"), FP4)
    for config in (gz.MX_CFG_SWAP_M32, gz.MX_CFG_SINGLE):
        d = torch.empty(m, n, device="cuda")
        gz.MxGated(m, n, k, FP4, torch.float32, activation=ACTS[act], config=config)(a, g, u, d, 1e6, 2.0 ** -6)
        want = np.where(np.arange(n) % 2 == 0, 64e6, -64e6 if act == "none" else 0.0)
        assert np.array_equal(d.cpu().double().numpy(), np.broadcast_to(want, (m, n)))


# ------------------------------------------------------------------------------------------- the checked build
def test_every_store_of_a_scale_is_checked_in_the_debug_build():
    """Each statement of the product kernels that writes into the scale array asks GZ_MX_SCALE_OK first."""
    text = (api.PKG / "csrc" / "mx_gemm.cuh").read_text().splitlines()
    stores = [i for i, line in enumerate(text) if "p.d_scales" in line]
    assert len(stores) == 3
    for i in stores:
        assert "GZ_MX_SCALE_OK" in text[i - 1] + text[i], text[i]


DEBUG_CHILD = """
import sys
sys.path.insert(0, {root!r})
import gemm_zoo_b200.api as api
api.lib_path = api.debug_lib_path  # before the first lib() call: this process runs the debug build
import gemm_zoo_b200 as gz
from tests import test_microscale_calls as t
for config, m, split in [(gz.MX_CFG_SWAP_M16, 13, 4), (gz.MX_CFG_SWAP_M64, 64, 8), (gz.MX_CFG_SINGLE, 130, 4), (gz.MX_CFG_PAIR, 300, 2)]:
    for out in t.FORMATS:
        t.test_quantised_gated_result_with_a_shared_k_range(t.NV, out, config, m, split)
print("DEBUG OK")
"""


@gpu
def test_debug_build_refuses_no_store_of_a_scale():
    import subprocess
    import sys
    from gemm_zoo_b200 import build as b
    b.build_lib(debug=True)
    r = subprocess.run([sys.executable, "-c", DEBUG_CHILD.format(root=str(api.PKG.parent))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "DEBUG OK" in r.stdout, (r.stdout[-500:], r.stderr[-2000:])


# ------------------------------------------------------------------------------------------- the allocator's stream
def _owner(t):
    """The stream whose pool a tensor's memory was taken from."""
    at = t.data_ptr()
    return [s["stream"] for s in torch.cuda.memory_snapshot() if s["address"] <= at < s["address"] + s["total_size"]]


@gpu
def test_memory_of_a_new_matrix_belongs_to_the_stream_that_writes_it():
    """Freed memory goes back to that stream's pool, where its next use is ordered behind the call that wrote it."""
    x = torch.randn(512, 4096, device="cuda")
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream, handle in ((side, side.cuda_stream), (side.cuda_stream, side.cuda_stream), (None, 0), (0, 0)):
        for current in (torch.cuda.default_stream(), side, other):
            with torch.cuda.stream(current):
                q = gz.mx_quantize(x, NV, stream=stream)
                assert _owner(q.codes) == [handle] and _owner(q.scales) == [handle]
                at, size = q.codes.data_ptr(), tuple(q.codes.shape)
                del q
            for s in (torch.cuda.default_stream(), side, other):  # freed: handed out again on its own stream alone
                with torch.cuda.stream(s):
                    again = torch.empty(size, dtype=torch.uint8, device="cuda")
                    assert (again.data_ptr() == at) <= (s.cuda_stream == handle)
                    del again
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------- nothing unreached
def test_every_function_of_the_microscaled_sources_is_called():
    import re
    files = [f for f in (api.PKG / "csrc").rglob("*") if f.suffix in (".cuh", ".cu", ".h")]
    text = "\n".join(f.read_text() for f in files)
    for f in files:
        if not f.name.startswith("mx_"):
            continue
        for name in re.findall(r"__device__ (?:__forceinline__|__noinline__)?\s*[\w:<>]+\s+(\w+)\(", f.read_text()):
            assert len(re.findall(rf"\b{name}\b", re.sub(r"//.*", "", text))) > 1, name


# ------------------------------------------------------------------------------------------- scales from elsewhere
def test_tile_scales_checks_its_arguments():
    ok = torch.zeros(3, 5, dtype=torch.uint8)
    for fmt in FORMATS:
        assert gz.tile_scales(ok, fmt).numel() == 1024
        assert gz.tile_scales(ok.view(torch.float8_e4m3fn), fmt).numel() == 1024
        for bad in (ok[0], ok[:, :, None], ok.half(), ok[:0], ok[:, :0]):
            with pytest.raises(ValueError):
                gz.tile_scales(bad, fmt)
    for fmt in (0, 3, 15, 18, None):
        with pytest.raises(ValueError):
            gz.tile_scales(ok, fmt)


# ------------------------------------------------------------------------------------------- limits of the split
@pytest.mark.parametrize("config,gated,most", [
    (gz.MX_CFG_PAIR, False, 4), (gz.MX_CFG_PAIR, True, 4), (gz.MX_CFG_SINGLE, False, 8), (gz.MX_CFG_SINGLE, True, 4),
    (gz.MX_CFG_PAIR_N128, False, 4), (gz.MX_CFG_SINGLE_N128, False, 4), (gz.MX_CFG_SWAP_M16, False, 8), (gz.MX_CFG_SWAP_M16, True, 8),
    (gz.MX_CFG_SWAP_M32, False, 8), (gz.MX_CFG_SWAP_M64, True, 8)])
def test_limits_of_the_split_are_those_of_the_header(config, gated, most):
    """A tile's output columns over 32 (row tiles), eight CTAs, and one part of K at least per CTA."""
    for split in (1, 2, 4, 8):
        for blocks in (1, 2, 3, 7, 8):
            d = gz.MxDesc.make(FP4, gz.DT_BF16, 16, 512, 256 * blocks, gated, config=config, split=split)
            assert (gz.mx_validate(d)[0] == api.GZ_OK) == (split <= most and split <= blocks)


# ------------------------------------------------------------------------------------------- lengths of one
@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("config", [gz.MX_CFG_AUTO, gz.MX_CFG_SWAP_M16, gz.MX_CFG_SWAP_M64, gz.MX_CFG_SINGLE, gz.MX_CFG_SINGLE_N128, gz.MX_CFG_PAIR,
                                    gz.MX_CFG_PAIR_N128])
def test_products_of_single_elements(fmt, config):
    for m, n, k in [(1, 1, 1), (1, 1, 2), (3, 1, 3), (1, 5, 1), (2, 2, 15), (1, 1, 257), (1, 129, 1)]:
        (a, av), (b, bv) = _mx(m, k, fmt, 1, True), _mx(n, k, fmt, 2, True)
        for dtype in (torch.float32, torch.float16):
            full, d = _out(m, n, n + 3, dtype)
            gz.MxGemm(m, n, k, fmt, dtype, ldd=n + 3, config=config)(a, b, None, d[:, :n], 1.0, 0.0)
            torch.cuda.synchronize()
            assert np.array_equal(d[:, :n].cpu().double().numpy(), av @ bv.T) and _guards_intact(full, m, n)
