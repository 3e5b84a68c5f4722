"""Microscaled 4-bit floats: the format against its definition (equal), the product against 64 bits.

Tolerance of the product: elements and scales are exact, so what is off is the accumulation in fp32 (K terms, each at most a step
of 2^-23 of the running sum, which the sum of the absolute products bounds) and the rounding to bf16 (2^-8 of the value for half a step).
"""
import pytest
import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def _reference(x):
    """(codes of the scales, values) by the definition, in 64 bits on the CPU: the nearest grid value, the even code at a tie."""
    b = x.detach().cpu().double().reshape(x.shape[0], x.shape[1] // 32, 32)
    amax = b.abs().amax(-1, keepdim=True)
    bad = ~b.isfinite().all(-1, keepdim=True)
    _, e = torch.frexp(torch.where(bad, 1.0, amax))
    e = torch.where(amax == 0, -127, (e - 3).clamp(min=-127)).double()
    v = torch.where(bad, 0.0, b) / torch.exp2(e)
    dist = (v.abs().unsqueeze(-1) - GRID).abs()
    low = dist.min(-1, keepdim=True).values
    near = dist == low
    even = near & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(-1, keepdim=True), even, near).to(torch.int8).argmax(-1)
    val = torch.where(bad, torch.nan, torch.copysign(GRID[code], v) * torch.exp2(e))
    return torch.where(bad, 255, e + 127).squeeze(-1).to(torch.uint8), val.flatten(1)


def _data(R, K, dt, seed=0):
    g = torch.Generator().manual_seed(seed + R * 7 + K)
    x = torch.randn(R, K, generator=g) * torch.exp2(torch.randint(-12, 12, (R, K // 32, 1), generator=g).float()).expand(R, K // 32, 32).reshape(R, K)
    return x.to(dt)


@pytest.mark.gpu
@pytest.mark.parametrize("R,K", [(1, 32), (3, 64), (31, 96), (128, 128), (129, 256), (257, 288), (40, 1184), (1000, 4096), (0, 64)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_and_read_back(R, K, dt):
    from nvshmem_b200.ops import mxfp4
    x = _data(R, K, dt).cuda()
    q = mxfp4.quantize_mxfp4(x)
    codes, val = _reference(x)
    assert q.shape == (R, K) and torch.equal(q.codes.cpu(), codes)
    assert torch.equal(q.dequantize(torch.float32).cpu().double(), val)
    assert torch.equal(q.dequantize().cpu(), val.to(torch.bfloat16)) and torch.equal(q.dequantize(torch.float16).cpu(), val.to(torch.float16))
    # bytes of rows and columns that do not exist are 0
    rb, kb, _ = q.scales.shape
    full = q.scales.view(rb, kb, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rb * 128, kb * 4)
    assert not full[R:].any() and not full[:, K // 32:].any()
    again = mxfp4.MxFp4.from_codes(q.data, q.codes)
    assert torch.equal(again.scales, q.scales) and torch.equal(again.data, q.data)


@pytest.mark.gpu
def test_every_border_and_its_neighbours():
    """Each border between two grid values, the floats next to it and the grid values themselves, in each binade and sign."""
    from nvshmem_b200.ops import mxfp4
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.999])
    near = torch.cat([border, torch.nextafter(border, torch.tensor(0.0)), torch.nextafter(border, torch.tensor(99.0))])
    row = torch.cat([near, torch.tensor([4.0, -0.0])])
    x = torch.stack([s * row * 2.0 ** e for e in (-120, -30, -1, 0, 1, 90) for s in (1.0, -1.0)])
    x[:, :30][x[:, :30].abs() >= x[:, 30:31].abs() * 2] = 0
    q = mxfp4.quantize_mxfp4(x.cuda())
    codes, val = _reference(x)
    assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.dequantize(torch.float32).cpu().double(), val)


@pytest.mark.gpu
def test_zeros_subnormals_and_bad_values():
    from nvshmem_b200.ops import mxfp4
    x = _data(8, 128, torch.float32)
    x[0] = 0
    x[1, :32] = 0
    x[2, :32] = torch.arange(32) * 2.0 ** -140           # subnormal: the scale is the smallest
    x[3, :32] = torch.finfo(torch.float32).max
    x[4, 40] = float("nan")
    x[5, 70] = float("inf")
    x[6, 0] = -float("inf")
    q = mxfp4.quantize_mxfp4(x.cuda())
    codes, val = _reference(x)
    assert torch.equal(q.codes.cpu(), codes)
    got = q.dequantize(torch.float32).cpu().double()
    assert torch.equal(got.isnan(), val.isnan()) and torch.equal(got.nan_to_num(), val.nan_to_num())


@pytest.mark.gpu
def test_strided_and_unaligned_rows():
    from nvshmem_b200.ops import mxfp4
    for dt in (torch.bfloat16, torch.float32):
        wide = _data(50, 320, dt).cuda()
        for cols in (slice(0, 96), slice(5, 101), slice(8, 296)):
            q = mxfp4.quantize_mxfp4(wide[::2, cols])
            want = mxfp4.quantize_mxfp4(wide[::2, cols].contiguous())
            assert torch.equal(q.data, want.data) and torch.equal(q.scales, want.scales)
        q = mxfp4.quantize_mxfp4(wide.t()[:, :32])
        want = mxfp4.quantize_mxfp4(wide.t()[:, :32].contiguous())
        assert torch.equal(q.data, want.data) and torch.equal(q.scales, want.scales)


def _check_product(x, w, out=None):
    from nvshmem_b200.ops import fused_gemm as fg
    from nvshmem_b200.ops import mxfp4
    xq, wq = mxfp4.quantize_mxfp4(x), mxfp4.quantize_mxfp4(w)
    got = mxfp4.gemm_mxfp4(xq, wq, out=out)
    torch.cuda.synchronize()
    fg.check_errors()
    xd, wd = xq.dequantize(torch.float32).double(), wq.dequantize(torch.float32).double()
    want, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    err = (got.double() - want).abs()
    lim = want.abs() * 2.0 ** -8 + mag * (x.shape[1] * 2.0 ** -23 if x.shape[1] < 4096 else 2.0 ** -11)
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    assert (err <= lim).all(), f"{int((err > lim).sum())} of {err.numel()} off, worst {(err / lim.clamp(min=1e-300)).max().item():.3g} of the tolerance"
    return got


@pytest.mark.gpu
def test_product_of_structured_operands():
    """Rows that pick one value of K each, with scales that differ by row and block: a wrong swizzle, descriptor or scale address shows."""
    from nvshmem_b200.ops import mxfp4
    for M, N, K in ((128, 256, 256), (256, 256, 512), (32, 128, 256), (64, 256, 512), (128, 128, 512), (300, 300, 416)):
        x, w = torch.zeros(M, K), torch.zeros(N, K)
        x[torch.arange(M), (torch.arange(M) * 37) % K] = torch.exp2((torch.arange(M) % 5 - 2).float())
        w += torch.tensor([1.0, 1.5, 2.0, 3.0, 4.0, 6.0])[(torch.arange(N)[:, None] + 3 * torch.arange(K)) % 6]
        w *= torch.exp2(((torch.arange(N)[:, None] * 5 + torch.arange(K) // 32 * 3) % 11 - 5).float())
        wq, xq = mxfp4.quantize_mxfp4(w.cuda()), mxfp4.quantize_mxfp4(x.cuda())
        want = xq.dequantize(torch.float32).double() @ wq.dequantize(torch.float32).double().t()
        assert torch.equal(mxfp4.gemm_mxfp4(xq, wq).double(), want), (M, N, K)   # one product a value: exact


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 16, 31, 33, 64, 65, 100, 128, 129, 257, 400])
@pytest.mark.parametrize("N,K", [(1, 32), (8, 64), (127, 288), (256, 256), (300, 1056), (513, 2048)])
def test_product_sizes(M, N, K):
    _check_product(_data(M, K, torch.bfloat16, 1).cuda(), _data(N, K, torch.bfloat16, 2).cuda())


# Products for each kernel, division of K, ragged edge and kind of store: (M, N, K) and the tile width and division that the rule takes on 148 SMs.
PLANS = [((5, 130, 4096), (32, 8)), ((32, 1000, 2560), (32, 4)), ((20, 9000, 2048), (32, 2)), ((17, 19001, 512), (32, 1)), ((7, 120, 8192), (32, 8)),
         ((50, 16001, 544), (64, 1)), ((130, 260, 4128), (64, 8)), ((300, 512, 8192), (64, 4)), ((129, 2043, 7168), (64, 2)),
         ((65, 8, 64), (64, 1)), ((190, 2100, 96), (64, 1)), ((3000, 4168, 96), (256, 1)), ((300, 4097, 1088), (128, 1)), ((1030, 1100, 2080), (128, 1)), ((500, 2047, 3200), (128, 1)),
         ((1024, 4096, 2048), (256, 1)), ((777, 8191, 1056), (256, 1)), ((2560, 4160, 544), (128, 1)), ((3000, 4160, 2080), (256, 1))]


def test_the_rule_takes_every_kernel():
    import ctypes
    from nvshmem_b200.ops import mxfp4
    out = (ctypes.c_int * 2)()
    got = []
    for shape, _ in PLANS:
        mxfp4._lib().bshmem_mxfp4_test_plan(*(ctypes.c_int64(v) for v in shape), 148, out)
        got.append((shape, tuple(out)))
    assert got == PLANS
    assert {c for _, (c, _) in got} == {32, 64, 128, 256} and {s for _, (_, s) in got} == {1, 2, 4, 8}


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [s for s, _ in PLANS])
def test_products_of_every_kernel(shape):
    M, N, K = shape
    w = _data(N, K, torch.bfloat16, 4).cuda()
    _check_product(_data(M, K, torch.bfloat16, 3).cuda(), w)
    # into the middle of a larger buffer: what lies around stays
    from nvshmem_b200.ops import mxfp4
    buf = torch.full((M + 2, N), 7.0, dtype=torch.bfloat16, device="cuda")
    x, wq = _data(M, K, torch.bfloat16, 3).cuda(), mxfp4.quantize_mxfp4(w)
    if N % 8 == 0:
        mxfp4.gemm_mxfp4(x, wq, out=buf[1:M + 1])
        assert (buf[0] == 7).all() and (buf[M + 1] == 7).all() and torch.equal(buf[1:M + 1], mxfp4.gemm_mxfp4(x, wq))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(16, 8192, 8192), (3, 7168, 2048), (512, 4096, 7168), (1500, 2816, 1984), (2048, 2047, 1024), (4100, 1032, 512), (2600, 1, 320), (5000, 9, 64), (1, 50001, 64),
                                   (9000, 9500, 96), (12345, 8712, 64), (9100, 300, 544)])
def test_larger_products(M, N, K):
    _check_product(torch.randn(M, K, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16),
                   torch.randn(N, K, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(torch.bfloat16) * 0.02)


@pytest.mark.gpu
def test_product_quantises_activations_and_fills_out():
    from nvshmem_b200.ops import mxfp4
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        x, w = _data(70, 256, dt).cuda(), mxfp4.quantize_mxfp4(_data(200, 256, dt, 9).cuda())
        buf = torch.full((72, 200), 7.0, dtype=torch.bfloat16, device="cuda")
        got = mxfp4.gemm_mxfp4(x, w, out=buf[1:71])
        assert torch.equal(got, mxfp4.gemm_mxfp4(mxfp4.quantize_mxfp4(x), w)) and got.data_ptr() == buf[1:].data_ptr()
        assert (buf[0] == 7).all() and (buf[71] == 7).all()


@pytest.mark.gpu
def test_bad_blocks_reach_only_their_rows():
    from nvshmem_b200.ops import mxfp4
    for M in (20, 200):
        x, w = torch.randn(M, 512, device="cuda"), torch.randn(300, 512, device="cuda")
        clean = mxfp4.gemm_mxfp4(x, mxfp4.quantize_mxfp4(w))
        x[3, 100], w[17, 400] = float("nan"), float("inf")
        got = mxfp4.gemm_mxfp4(x, mxfp4.quantize_mxfp4(w))
        assert got[3].isnan().all() and got[:, 17].isnan().all()
        keep = torch.ones_like(got, dtype=torch.bool)
        keep[3], keep[:, 17] = False, False
        assert torch.equal(got[keep], clean[keep])


@pytest.mark.gpu
def test_empty_products():
    from nvshmem_b200.ops import mxfp4
    x, w = torch.zeros(0, 64, device="cuda"), mxfp4.quantize_mxfp4(torch.ones(5, 64, device="cuda"))
    assert mxfp4.gemm_mxfp4(x, w).shape == (0, 5)
    assert mxfp4.gemm_mxfp4(torch.ones(3, 64, device="cuda"), mxfp4.quantize_mxfp4(x)).shape == (3, 0)


def test_codes_and_scale_order_agree_with_the_definition():
    """The order of the scales, on the CPU: byte (r % 32) * 16 + (r / 32) * 4 + s of block (r / 128, k / 128)."""
    from nvshmem_b200.ops.mxfp4 import MxFp4
    R, S = 300, 9
    codes = torch.randint(0, 256, (R, S), dtype=torch.uint8)
    q = MxFp4.from_codes(torch.zeros(R, S * 16, dtype=torch.uint8), codes)
    assert q.shape == (R, S * 32) and tuple(q.scales.shape) == (3, 4, 512) and torch.equal(q.codes, codes)
    for r, s in ((0, 0), (31, 3), (32, 0), (127, 8), (128, 4), (299, 8)):
        assert q.scales[r // 128, s // 4, (r % 32) * 16 + r % 128 // 32 * 4 + s % 4] == codes[r, s]


def test_refusals():
    from nvshmem_b200.ops.fused_gemm import FusedGemmError
    from nvshmem_b200.ops.mxfp4 import gemm_mxfp4, MxFp4, quantize_mxfp4
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)
    q = MxFp4(u8(4, 32), u8(1, 2, 512), (4, 64))
    bad = [lambda: quantize_mxfp4(torch.zeros(4, 33)), lambda: quantize_mxfp4(torch.zeros(4, 0)), lambda: quantize_mxfp4(torch.zeros(64)),
           lambda: quantize_mxfp4(torch.zeros(4, 64).double()), lambda: quantize_mxfp4(torch.zeros(4, 64)), lambda: MxFp4(u8(4, 32), u8(1, 2, 512), (5, 64)),
           lambda: MxFp4(u8(4, 32), u8(1, 1, 512), (4, 64)), lambda: MxFp4(u8(4, 24), u8(1, 2, 512), (4, 48)), lambda: MxFp4.from_codes(u8(4, 32), u8(4, 3)),
           lambda: gemm_mxfp4(q, torch.zeros(4, 64)), lambda: gemm_mxfp4(q, MxFp4(u8(4, 16), u8(1, 2, 512), (4, 32))), lambda: gemm_mxfp4(q, q), lambda: q.dequantize(torch.int8),
           lambda: q.dequantize()]
    for call in bad:
        with pytest.raises(FusedGemmError):
            call()


def test_limits_of_the_entry_points():
    """Sizes that a launch cannot take are refused before anything is launched (or looked at)."""
    import ctypes
    from nvshmem_b200.ops import mxfp4
    lib = mxfp4._lib()
    for R, K in ((1, 1 << 26), (1, (1 << 26) + 32), (1, 33), (1, 0), (-1, 32), (1 << 31, 32)):
        assert lib.bshmem_mxfp4_quantize(None, 0, R, K, K, None, None, None) == 2
        assert lib.bshmem_mxfp4_dequantize(None, None, R, K, 0, None, None) == 2
        a = mxfp4._GemmArgs(M=R, N=8, K=K)
        assert lib.bshmem_mxfp4_gemm(ctypes.byref(a), None) == 2
    assert lib.bshmem_mxfp4_quantize(None, 0, 1, (1 << 26) - 32, 0, None, None, None) == 1   # the size would do
    assert lib.bshmem_mxfp4_quantize(None, 0, 0, 32, 32, None, None, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_the_longest_rows(dt):
    """K up to the limit: a row gives the bytes of the same blocks laid out as shorter rows."""
    from nvshmem_b200.ops import mxfp4
    for K, rows in (((1 << 26) - 32, 337), ((1 << 26) - 1024, 340), (65535 * 1024 + 32, 169)):   # divisors of K / 32
        assert K % (rows * 32) == 0
        x = torch.randn(1, K, device="cuda", generator=torch.Generator("cuda").manual_seed(rows)).to(dt)
        q, short = mxfp4.quantize_mxfp4(x), mxfp4.quantize_mxfp4(x.view(rows, K // rows))
        assert torch.equal(q.data.view(-1), short.data.view(-1)) and torch.equal(q.codes.view(-1), short.codes.view(-1))
        assert not q.scales.view(-1, 32, 4, 4)[:, 1:].any() and not q.scales.view(-1, 32, 4, 4)[:, :, 1:].any()   # rows past the end
        assert torch.equal(q.dequantize().view(-1), short.dequantize().view(-1))
        # a product that picks values of both ends: exact
        pick = torch.zeros(2, K, device="cuda", dtype=dt)
        pick[0, 5], pick[1, K - 3] = 1.0, 2.0
        got = mxfp4.gemm_mxfp4(pick, q)
        values = q.dequantize(torch.float32)
        assert torch.equal(got.float(), torch.stack([values[:, 5], 2 * values[:, K - 3]]).to(torch.bfloat16).float())


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 256, 8192), (16, 1000, 8192), (33, 520, 4096), (64, 8192, 8192), (130, 260, 12288), (300, 512, 8192), (512, 4096, 7168), (777, 1040, 5024),
                                   (1024, 4096, 4096), (2048, 2047, 8192)])
def test_long_sums_are_exact_where_fp32_is(M, N, K):
    """Elements of the grid with one scale per row: every product is a multiple of 1/4 of the rows' scales and every sum of them below 36 K / 4 <= 2^21
    multiples, so that fp32 holds all of them and the result is the exact sum, rounded once."""
    from nvshmem_b200.ops import mxfp4
    g = torch.Generator(device="cuda").manual_seed(M)

    def operand(R):
        v = GRID.to("cuda")[torch.randint(0, 8, (R, K), generator=g, device="cuda")] * (torch.randint(0, 2, (R, K), generator=g, device="cuda") * 2 - 1)
        v[:, ::32] = 6.0   # every block has the same scale before the row's own
        return v.float() * torch.exp2(torch.randint(-3, 4, (R, 1), generator=g, device="cuda").float())

    x, w = operand(M), operand(N)
    xq, wq = mxfp4.quantize_mxfp4(x), mxfp4.quantize_mxfp4(w)
    assert torch.equal(xq.dequantize(torch.float32), x) and torch.equal(wq.dequantize(torch.float32), w)
    assert torch.equal(mxfp4.gemm_mxfp4(xq, wq), (x.double() @ w.double().t()).to(torch.bfloat16))
