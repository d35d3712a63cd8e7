"""4-bit linear layers on the GPU against 64-bit products of the same codes.

Tolerance. With u = 2^-24 the kernel's fp32 sum of a group of at most 128 inputs
passes at most 32 + 4 roundings (a matrix instruction's 32 products, four
instructions) on terms of at most |x| (128 + 15) s for the codes and as much
again for the offset's product; the groups' sums and the waves' add at most
K / 32 + 12 roundings on partial sums of at most sum |x (c - z)| s. Then one
rounding to the output type, half a step: eps / 2 of the value."""

import pytest
import torch

from qsa_vllm_amd.ops import int4_linear, int4_pack, int4_quantize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _weight(gen, n, k, group, dtype, zeros, scale=0.01):
    groups = -(-k // group)
    codes = torch.randint(0, 16, (n, k), generator=gen, dtype=torch.uint8)
    scales = ((torch.rand(n, groups, generator=gen) + 0.5) * scale).to(dtype)
    z = torch.randint(0, 16, (n, groups), generator=gen, dtype=torch.uint8) if zeros else None
    return codes, scales, z


def _want(x, codes, scales, zeros, group, bias=None):
    """(result, tolerance) in 64 bits."""
    k = codes.shape[1]
    s = scales.double().repeat_interleave(group, 1)[:, :k]
    z = (zeros.double() if zeros is not None else torch.full_like(scales, 8, dtype=torch.float64))
    w = (codes.double() - z.repeat_interleave(group, 1)[:, :k]) * s
    xd = x.double()
    y = xd @ w.t()
    sums = U * (36 * 2 * 143 * (xd.abs() @ s.t()) + (k / 32 + 12) * (xd.abs() @ w.abs().t()))
    if bias is not None:
        y = y + bias.double()
        sums = sums + U * y.abs()
    # the smallest subnormal's half step, for fp16 results near zero
    return y, sums + (torch.finfo(x.dtype).eps / 2) * (y.abs() + sums) + 2.0 ** -25


def _check(got, want):
    y, tol = want
    off = (got.cpu().double() - y).abs()
    assert (off <= tol).all(), f"{(off / tol).max().item():.2f} times the tolerance"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,n,k,zeros", [
    (1, 256, 512, False), (1, 17, 8, True), (2, 1, 128, True), (3, 100, 1000, True),
    (15, 33, 264, False), (16, 48, 2048, True), (17, 64, 640, True), (31, 80, 4096, False),
    (33, 96, 136, True), (61, 130, 1536, True), (64, 31, 256, False), (65, 47, 384, True),
    (130, 64, 520, True), (250, 272, 1024, True), (300, 40, 96, False), (5, 2100, 256, False),
    (9, 16, 5632, True)])
def test_matches_64_bits(rows, n, k, zeros, group, dtype):
    gen = torch.Generator().manual_seed(rows * 1000 + n + k)
    codes, scales, z = _weight(gen, n, k, group, dtype, zeros)
    x = torch.randn(rows, k, generator=gen).to(dtype)
    bias = torch.randn(n, generator=gen).to(dtype) if zeros else None
    w = int4_pack(codes.to(DEV), scales.to(DEV), z.to(DEV) if zeros else None, group_size=group)
    got = int4_linear(x.to(DEV), w, bias.to(DEV) if zeros else None)
    assert got.dtype == dtype and got.shape == (rows, n)
    _check(got, _want(x, codes, scales, z, group, bias))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 7, 20, 64, 200])
@pytest.mark.parametrize("k,group", [(1, 32), (7, 64), (129, 128), (333, 32), (1023, 64)])
def test_whole_numbers_are_exact(rows, k, group, dtype):
    """Small whole activations, scales of powers of two: every sum is exact in
    fp32, so the result is the exact value rounded once. Any width."""
    gen = torch.Generator().manual_seed(k + rows)
    n = 37
    codes = torch.randint(0, 16, (n, k), generator=gen, dtype=torch.uint8)
    groups = -(-k // group)
    scales = (2.0 ** torch.randint(-3, 1, (n, groups), generator=gen).float()).to(dtype)
    z = torch.randint(0, 16, (n, groups), generator=gen, dtype=torch.uint8)
    x = torch.randint(-2, 3, (rows, k), generator=gen).to(dtype)
    w = int4_pack(codes.to(DEV), scales.to(DEV), z.to(DEV), group_size=group)
    got = int4_linear(x.to(DEV), w)
    exact, _ = _want(x, codes, scales, z, group)
    assert torch.equal(got.cpu(), exact.float().to(dtype))


# Every block shape of the kernel for more than 16 rows, by what is least of
# rows and outputs: 32 x 32, 32 x 64, 32 x 96, 64 x 128 and 64 x 192, each with odd ends.
BLOCKS = [(40, 500), (100, 2100), (204, 1544), (64, 9000), (50, 49500), (250, 22500)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,n", BLOCKS)
def test_block_shapes_are_exact_on_whole_numbers(rows, n, group, zeros, dtype):
    """Fewer k tiles than the waves share, and a short last one: 128 to 1288 inputs."""
    gen = torch.Generator(device=DEV).manual_seed(rows + n)
    for k in (128, 520, 1288):
        codes = torch.randint(0, 16, (n, k), generator=gen, device=DEV, dtype=torch.uint8)
        groups = -(-k // group)
        scales = (2.0 ** torch.randint(-3, 1, (n, groups), generator=gen, device=DEV).float()).to(dtype)
        z = torch.randint(0, 16, (n, groups), generator=gen, device=DEV, dtype=torch.uint8) if zeros else None
        x = torch.randint(-2, 3, (rows, k), generator=gen, device=DEV).to(dtype)
        got = int4_linear(x, int4_pack(codes, scales, z, group_size=group))
        s = scales.float().repeat_interleave(group, 1)[:, :k]
        shift = z.float().repeat_interleave(group, 1)[:, :k] if zeros else 8.0
        # whole multiples of 2^-3 below 2^17: exact in fp32 in any order
        exact = x.float() @ ((codes.float() - shift) * s).t()
        assert torch.equal(got, exact.to(dtype)), k


def test_strides_alignment_and_out():
    gen = torch.Generator().manual_seed(3)
    n, k, group, dtype = 50, 256, 64, torch.bfloat16
    codes, scales, z = _weight(gen, n, k, group, dtype, True)
    w = int4_pack(codes.to(DEV), scales.to(DEV), z.to(DEV), group_size=group)
    for offset, stride in ((0, 256), (1, 256), (8, 264), (3, 301), (0, 261)):
        big = torch.randn(6 * stride + 300, generator=gen).to(dtype)
        x = big.as_strided((5, k), (stride, 1), offset)
        want = _want(x, codes, scales, z, group)
        _check(int4_linear(big.to(DEV).as_strided((5, k), (stride, 1), offset), w), want)
        out = torch.full((7, 99), 7.0, dtype=dtype, device=DEV)
        assert int4_linear(x.to(DEV), w, out=out[1:6, 5:55]).data_ptr() == out[1, 5:].data_ptr()
        _check(out[1:6, 5:55], want)
        keep = out.clone()
        keep[1:6, 5:55] = 7.0
        assert (keep == 7.0).all()                      # nothing beside the result is written
    one = torch.randn(1, k, generator=gen).to(dtype)
    want = _want(one.expand(4, k), codes, scales, z, group)
    _check(int4_linear(one.to(DEV).expand(4, k), w), want)      # the same row four times
    x3 = torch.randn(2, 3, k, generator=gen).to(dtype)
    got = int4_linear(x3.to(DEV), w)
    assert got.shape == (2, 3, n)
    _check(got.view(6, n), _want(x3.view(6, k), codes, scales, z, group))
    assert int4_linear(x3[0, 0].to(DEV), w).shape == (n,)
    assert int4_linear(x3[:, :0].to(DEV), w).shape == (2, 0, n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_far_apart(dtype):
    """Offsets of a block's rows past 32 bits, taken element by element (an odd
    distance) or not (a distance that 32 bits do not hold)."""
    if torch.cuda.mem_get_info()[0] < (30 << 30):
        pytest.skip("needs 30 GiB")
    gen = torch.Generator().manual_seed(12)
    codes, scales, z = _weight(gen, 40, 200, 64, dtype, True)
    w = int4_pack(codes.to(DEV), scales.to(DEV), z.to(DEV), group_size=64)
    x = torch.randn(20, 200, generator=gen).to(dtype)
    for far in ((1 << 29) + 1, 1 << 29):
        store = torch.empty(19 * far + 200, dtype=dtype, device=DEV)
        view = store.as_strided((20, 200), (far, 1))
        view.copy_(x)
        for rows in (1, 16, 20):
            _check(int4_linear(view[:rows], w), _want(x[:rows], codes, scales, z, 64))
        del store, view


def test_rows_do_not_touch_each_other():
    """A row of NaN or infinities leaves the others' bits alone, and a row's bits
    do not depend on its place or on what is past the last row."""
    gen = torch.Generator().manual_seed(4)
    for dtype in (torch.bfloat16, torch.float16):
        codes, scales, z = _weight(gen, 64, 512, 64, dtype, True)
        w = int4_pack(codes.to(DEV), scales.to(DEV), z.to(DEV), group_size=64)
        x = torch.randn(20, 512, generator=gen).to(dtype).to(DEV)
        clean = int4_linear(x, w)
        dirty = x.clone()
        dirty[3] = float("nan")
        dirty[17, 100] = float("inf")
        got = int4_linear(dirty, w)
        rest = [r for r in range(20) if r not in (3, 17)]
        assert torch.equal(got[rest], clean[rest])
        assert got[3].isnan().all() and not got[17].isfinite().any()


def test_repeated_calls_give_the_same_bits_and_graphs_replay():
    gen = torch.Generator().manual_seed(5)
    codes, scales, z = _weight(gen, 1000, 2048, 128, torch.bfloat16, False)
    w = int4_pack(codes.to(DEV), scales.to(DEV), group_size=128)
    for rows in (1, 40, 100):
        x = torch.randn(rows, 2048, generator=gen).bfloat16().to(DEV)
        first = int4_linear(x, w)
        buf, out = x.clone(), torch.empty_like(first)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            assert torch.equal(int4_linear(x, w), first)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            int4_linear(buf, w, out=out)
        for step in range(3):
            buf.copy_(x * (step + 1))
            graph.replay()
            want = int4_linear(buf.clone(), w)
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_a_weight_past_2_gib_of_codes():
    """Byte offsets past 32 bits: only the last outputs are compared."""
    n, k = 300000, 16384                      # 2.46 GB of codes
    free = torch.cuda.mem_get_info()[0]
    if free < (24 << 30):
        pytest.skip("needs 24 GiB of free GPU memory")
    gen = torch.Generator(device=DEV).manual_seed(6)
    codes = torch.randint(0, 16, (n, k), generator=gen, device=DEV, dtype=torch.uint8)
    scales = torch.full((n, k // 128), 0.01, dtype=torch.bfloat16, device=DEV)
    w = int4_pack(codes, scales)
    x = torch.randn(2, k, generator=gen, device=DEV).bfloat16()
    got = int4_linear(x, w)
    last = slice(n - 40, n)
    _check(got[:, last], _want(x.cpu(), codes[last].cpu(), scales[last].cpu(), None, 128))
    _check(got[:, :40], _want(x.cpu(), codes[:40].cpu(), scales[:40].cpu(), None, 128))


def test_quantized_layer_is_near_its_weight():
    """The layer on a rounded weight equals the product with the weight that
    dequantize() gives, whose distance from the original is tested on the CPU."""
    gen = torch.Generator().manual_seed(7)
    weight = (torch.randn(200, 600, generator=gen) * 0.02).bfloat16()
    x = torch.randn(4, 600, generator=gen).bfloat16()
    for zero_points in (False, True):
        q = int4_quantize(weight.to(DEV), group_size=64, zero_points=zero_points)
        y = x.double() @ q.dequantize().cpu().double().t()
        scale = q.scales.float().max().item()
        tol = U * (36 * 286 * scale * x.double().abs().sum(1, keepdim=True)
                   + 31 * (x.double().abs() @ q.dequantize().cpu().double().abs().t()))
        off = (int4_linear(x.to(DEV), q).cpu().double() - y).abs()
        assert (off <= tol + 2.0 ** -8 * (y.abs() + tol)).all()


def test_refusals():
    gen = torch.Generator().manual_seed(8)
    codes, scales, _ = _weight(gen, 32, 128, 128, torch.bfloat16, False)
    w = int4_pack(codes.to(DEV), scales.to(DEV))
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device=DEV)
    bias = torch.zeros(32, dtype=torch.bfloat16, device=DEV)
    for bad, match in ((lambda: int4_linear(x.half(), w), "scales"),
                       (lambda: int4_linear(x.float(), w), "bf16 or fp16"),
                       (lambda: int4_linear(x[:, :64], w), "columns"),
                       (lambda: int4_linear(x.t().contiguous().t(), w), "unit column"),
                       (lambda: int4_linear(x, w, bias[:31]), "bias"),
                       (lambda: int4_linear(x, w, bias.float()), "bias"),
                       (lambda: int4_linear(x.cpu(), w), "GPU|device|backend"),
                       (lambda: int4_linear(x, w, out=x[:, :32].float()), "out"),
                       (lambda: int4_linear(x, w, out=x[:1, :32].expand(2, 32)), "overlapping"),
                       (lambda: int4_linear(x, w, out=x[:1, :32]), "out must be")):
        with pytest.raises(RuntimeError, match=match):
            bad()
    assert int4_linear(x[:0], w).shape == (0, 32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros,group", [(True, 32), (False, 128), (True, 64)])
@pytest.mark.parametrize("rows,k,offset", [(1, 512, 0), (3, 200, 0), (7, 264, 0), (16, 1023, 0), (20, 200, 0),
                                           (61, 520, 0), (250, 392, 0), (5, 200, 1), (40, 72, 1)])
def test_infinite_and_huge_activations(rows, k, offset, zeros, group, dtype):
    """What x times the dequantized weight gives in any order: an infinity where
    one is met by weights of one sign, NaN by 0 or by unlike signs, and finite sums of
    bf16 values whose product with the codes alone would overflow. In rows of
    every kind: sixteen bytes at a time or not, a width that is no whole tile."""
    gen = torch.Generator().manual_seed(rows + k)
    n = 4200 if rows in (7, 250) else 70
    codes, scales, z = _weight(gen, n, k, group, dtype, zeros)
    x = torch.randn(rows, k, generator=gen).to(dtype)
    special = {0: [(0, "inf")], 2: [(k - 1, "-inf")], 3: [(5, "inf"), (k // 2, "inf")],
               4: [(1, "inf"), (9, "-inf")], 6: [(k - 2, "nan")], 17: [(3, "-inf")], 19: [(k // 3, "nan")],
               33: [(k - 9, "inf")], 60: [(0, "inf")], 200: [(63, "-inf")], 249: [(k - 1, "inf")]}
    for row, places in special.items():
        if row < rows:
            for at, value in places:
                x[row, at] = float(value)
    huge = [r for r in range(rows) if r % 5 == 1] if dtype == torch.bfloat16 else []
    for r in huge:
        x[r] = (x[r].float() * 2.0 ** 119).bfloat16()
    w = int4_pack(codes.to(DEV), scales.to(DEV), z.to(DEV) if zeros else None, group_size=group)
    store = torch.zeros(rows * (k + 8) + 8, dtype=dtype, device=DEV)
    view = store.as_strided((rows, k), (k + 8 - k % 8, 1), offset)
    view.copy_(x)
    got = int4_linear(view, w).cpu().double()
    wd = w.dequantize().cpu().double()
    for r in range(rows):
        terms = x[r].double() * wd
        want = terms.sum(1)
        if r in special:
            assert not torch.isfinite(want).all()
            assert torch.equal(torch.nan_to_num(got[r], nan=7.0), torch.nan_to_num(want, nan=7.0)), r
        else:
            s = scales.double().repeat_interleave(group, 1)[:, :k]
            sums = U * (36 * 2 * 143 * (x[r].double().abs() * s).sum(1) + (k + 12) * terms.abs().sum(1))
            tol = sums + torch.finfo(dtype).eps / 2 * (want.abs() + sums) + 2.0 ** -25
            assert ((got[r] - want).abs() <= tol).all(), r


def test_a_nan_row_ends_at_once():
    """Rows of NaN, as padding may hold them, cost little more than others."""
    gen = torch.Generator(device=DEV).manual_seed(40)
    weight = (torch.randn(11264, 4096, generator=gen, device=DEV) * 0.02).bfloat16()
    w = int4_quantize(weight)
    x = torch.randn(61, 4096, generator=gen, device=DEV).bfloat16()
    dirty = x.clone()
    dirty[20:] = float("nan")
    out = torch.empty(61, 11264, dtype=torch.bfloat16, device=DEV)
    times = {}
    for name, rows in (("clean", x), ("dirty", dirty)):
        for _ in range(8):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(10):
                int4_linear(rows, w, out=out)
            b.record()
            b.synchronize()
            times[name] = min(times.get(name, 1e9), a.elapsed_time(b))
    assert out[20:].isnan().all() and torch.isfinite(out[:20]).all()
    assert times["dirty"] < 4 * times["clean"], times


@pytest.mark.parametrize("rows,n,dtype", [(1 << 20, 4096, torch.bfloat16), (150000, 99072, torch.float16)])
def test_millions_of_blocks(rows, n, dtype):
    """Launches of many blocks, to the last row and output."""
    k = 128
    if torch.cuda.mem_get_info()[0] < (64 << 30):
        pytest.skip("needs 64 GiB of free GPU memory")
    gen = torch.Generator(device=DEV).manual_seed(rows)
    codes = torch.randint(0, 16, (n, k), generator=gen, device=DEV, dtype=torch.uint8)
    scales = torch.full((n, 1), 0.125, dtype=dtype, device=DEV)
    w = int4_pack(codes, scales)
    x = torch.randint(-2, 3, (rows, k), generator=gen, device=DEV, dtype=torch.int8).to(dtype)
    got = int4_linear(x, w)
    weight = w.dequantize()
    for part in (slice(0, 70), slice(rows // 2, rows // 2 + 70), slice(rows - 70, rows)):
        # multiples of 2^-3 below 2^12: exact in fp32 in any order
        assert torch.equal(got[part], (x[part].float() @ weight.t()).to(dtype))
