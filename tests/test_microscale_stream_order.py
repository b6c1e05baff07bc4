"""Stream order between consecutive launches of the microscaled operators, without host synchronisation: what one call
writes the next one reads, and buffers are written again while later launches are already resident.  Every result is kept
and compared bit for bit with the same call made with a device synchronisation around it."""
import pytest
import torch

import gemm_zoo_b200 as gz
from tests.test_microscale import FP4, NV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [FP4, NV])
@pytest.mark.parametrize("layout", [gz.ROW_MAJOR, gz.COL_MAJOR])
@pytest.mark.parametrize("rows,k", [(1, 64), (1, 4096), (33, 512), (256, 4096), (3000, 1000)])
def test_codes_and_scales_written_again_and_again(fmt, layout, rows, k):
    """Quantise x_i and decode it, all through one pair of buffers; scales differ from call to call."""
    steps = 60
    shape = (rows, k) if layout == gz.ROW_MAJOR else (k, rows)
    xs = [torch.randn(shape, device="cuda").mul_(2.0 ** (i % 7 - 3)).bfloat16() for i in range(6)]
    want = []
    for x in xs:
        q = gz.mx_quantize(x, fmt, layout=layout)
        torch.cuda.synchronize()
        want.append(gz.mx_dequantize(q, torch.empty_like(x), layout=layout))
        torch.cuda.synchronize()
    q = gz.MxMatrix.empty(rows, k, fmt)
    ys = [torch.empty_like(xs[0]) for _ in range(steps)]
    torch.cuda.synchronize()

    def run(stream):
        for i, y in enumerate(ys):
            gz.mx_quantize(xs[i % 6], fmt, layout=layout, out=q, stream=stream)
            gz.mx_dequantize(q, y, layout=layout, stream=stream)

    run(None)
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 6]) for i, y in enumerate(ys))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(torch.cuda.current_stream())
    for _ in range(3):
        for y in ys:
            y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[i % 6]) for i, y in enumerate(ys))


@pytest.mark.parametrize("config,m", [(gz.MX_CFG_SWAP_M16, 16), (gz.MX_CFG_SWAP_M64, 64), (gz.MX_CFG_SINGLE_N128, 200), (gz.MX_CFG_PAIR, 256)])
def test_epilogue_vectors_written_by_the_call_before(config, m):
    """bias, row and column scales come out of a decode that the product follows directly."""
    n, k, steps = 384, 512, 40
    a, b = (gz.mx_quantize(torch.randn(r, k, device="cuda"), NV) for r in (m, n))
    plan = gz.MxGemm(m, n, k, NV, torch.float32, config=config)
    vectors = [gz.mx_quantize(torch.randn(3, max(m, n), device="cuda") * 2.0 ** i, NV) for i in range(4)]
    v = torch.empty(3, max(m, n), device="cuda")
    d = [torch.empty(m, n, device="cuda") for _ in range(steps)]

    def step(i, out, stream=None):
        gz.mx_dequantize(vectors[i % 4], v, stream=stream)
        plan(a, b, None, out, 0.125, 0.0, bias=v[0, :n], row_scale=v[1, :m], col_scale=v[2, :n], stream=stream)

    want = []
    for i in range(4):
        torch.cuda.synchronize()
        want.append(torch.empty(m, n, device="cuda"))
        gz.mx_dequantize(vectors[i], v)
        torch.cuda.synchronize()
        plan(a, b, None, want[i], 0.125, 0.0, bias=v[0, :n], row_scale=v[1, :m], col_scale=v[2, :n])
        torch.cuda.synchronize()
    assert not torch.equal(want[0], want[1])
    for i, out in enumerate(d):
        step(i, out)
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i % 4]) for i, out in enumerate(d))


@pytest.mark.parametrize("config,m", [(gz.CFG_SWAP_M16, 16), (gz.CFG_1CTA_N64, 128), (gz.CFG_2CTA_N256, 256)])
def test_bias_of_a_16_bit_product_written_by_the_product_before(config, m):
    """A one-row fp32 product gives the bias of the next product; both launches may be resident together."""
    n, k, steps = 512, 256, 40
    a, w = torch.randn(m, k, device="cuda").bfloat16(), torch.randn(n, k, device="cuda").bfloat16()
    rows = [torch.randn(1, k, device="cuda").bfloat16() for _ in range(4)]
    first = gz.Plan(gz.GemmDesc.make(gz.DT_BF16, gz.DT_F32, 1, n, k, gz.ROW_MAJOR, gz.COL_MAJOR))
    second = gz.Plan(gz.GemmDesc.make(gz.DT_BF16, gz.DT_F32, m, n, k, gz.ROW_MAJOR, gz.COL_MAJOR, config=config))
    v = torch.empty(1, n, device="cuda")
    want = []
    for r in rows:
        first.run(r, w, None, v, 1.0, 0.0)
        torch.cuda.synchronize()
        want.append(torch.empty(m, n, device="cuda"))
        second.run_ex(a, w, None, want[-1], 1.0, 0.0, bias=v.view(-1))
        torch.cuda.synchronize()
    d = [torch.empty(m, n, device="cuda") for _ in range(steps)]
    for i, out in enumerate(d):
        first.run(rows[i % 4], w, None, v, 1.0, 0.0)
        second.run_ex(a, w, None, out, 1.0, 0.0, bias=v.view(-1))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i % 4]) for i, out in enumerate(d))


@pytest.mark.parametrize("config,m,split", [(gz.MX_CFG_AUTO, 1, 0), (gz.MX_CFG_SWAP_M64, 40, 8), (gz.MX_CFG_SINGLE, 130, 4), (gz.MX_CFG_PAIR, 300, 2),
                                            (gz.MX_CFG_PAIR, 2500, 1)])
def test_repeated_calls_give_the_same_bits(config, m, split):
    """Sums are taken in one order whatever runs when: a feed-forward layer of arbitrary values, again and again."""
    n, k = 640, 2048
    x = torch.randn(m, k, device="cuda").bfloat16()
    g, u, w = (gz.mx_quantize(torch.randn(s, device="cuda") * 5, NV) for s in ((n, k), (n, k), (k, n)))
    q, h = gz.MxMatrix.empty(m, k, NV), gz.MxMatrix.empty(m, n, NV)
    gated, down = gz.MxGated(m, n, k, NV, NV, config=config, split=split), gz.MxGemm(m, k, n, NV, torch.float32)
    y = [torch.empty(m, k, device="cuda") for _ in range(12)]
    codes, scales = [], []
    for out in y:
        gz.mx_quantize(x, NV, out=q)
        gated(q, g, u, h, 0.02, 0.02)
        down(h, w, None, out, 0.02, 0.0)
        codes.append(h.codes.clone())
        scales.append(h.scales.clone())
    torch.cuda.synchronize()
    assert float(y[0].abs().max()) > 0
    for got in (y, codes, scales):
        assert all(torch.equal(v, got[0]) for v in got)
