"""GPU: int8 rows and W8A8 products against their definition in 64 bits."""
import pytest
import torch

from mini_qwen_b200.kernels import (moe_permute_plan, quantize_rows_int8, w8a8_gemm, w8a8_grouped_gemm, w8a8_grouped_swiglu,
                                    w8a8_grouped_swiglu_gather)
from mini_qwen_b200.model.layers import LinearW8A8
from mini_qwen_b200.quantization import quantize_channels_int8
import w8a8_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def hidden(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def weight(g, *shape):
    q = torch.randint(-128, 128, shape, generator=g, device=DEV, dtype=torch.int8)
    return q, torch.rand(shape[:-1], generator=g, device=DEV) * 0.01 + 1e-4


def offsets(counts, dtype=torch.int32):
    return torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=dtype, device=DEV)


# ---- rows ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(1, 1), (3, 7), (9, 16), (8, 64), (5, 260), (33, 768), (2, 2048), (7, 4096), (3, 4104),
                                    (2, 8192), (1, 20001)])
def test_rows_are_quantised_as_defined(dtype, rows, K):
    x = hidden(gen(rows * K), rows, K, dtype=dtype) * 3
    q, s = quantize_rows_int8(x)
    rq, rs = R.quantize(x)
    assert q.dtype == torch.int8 and s.dtype == torch.float32
    assert torch.equal(s.double(), rs) and torch.equal(q.double(), rq)
    cq, cs = quantize_channels_int8(x)                # the weights' quantiser does the same
    assert torch.equal(q, cq) and torch.equal(s, cs)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quotients_that_are_halves_go_to_even(dtype):
    x = torch.zeros(4, 256, device=DEV)
    x[0, 1:] = torch.arange(255, device=DEV) / 2 - 63.5          # scale 1: halves
    x[0, 0] = 127
    x[1] = x[0] * 3                                              # scale 3: 1/3 is not representable, the halves are still halves
    x[2] = x[0] * 2.0 ** -12
    x[3] = -x[0]
    x = x.to(dtype)
    q, s = quantize_rows_int8(x)
    rq, rs = R.quantize(x)
    assert torch.equal(q.double(), rq) and torch.equal(s.double(), rs)


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_rows(dtype):
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    x = torch.zeros(9, 40, device=DEV, dtype=dtype)
    x[1, 3] = top
    x[2, 3], x[2, 4] = -top, top / 2
    x[3] = tiny                                                  # all the smallest subnormal
    x[4, 0], x[4, 1] = tiny * 5, -tiny
    x[5, 7] = float("inf")
    x[6, 39] = float("nan")
    x[7, 0], x[7, 1], x[7, 2] = float("nan"), float("-inf"), 1
    x[8, 0] = 1
    q, s = quantize_rows_int8(x)
    rq, rs = R.quantize(x)
    assert torch.equal(torch.isnan(s), torch.isnan(rs)) and torch.isnan(s).sum() == 3
    assert torch.equal(s.nan_to_num().double(), rs.nan_to_num()) and torch.equal(q.double(), rq)
    assert s[0] == 0 and not q[0].any()


def test_rows_of_a_wider_tensor_are_read_in_place():
    g = gen(3)
    base = hidden(g, 20, 100)
    for x in (base[:, 4:68], base[::3, 1:65], base[:, 8:72][5:6], base.t(), base[2].expand(4, 100), base[0],
              base.view(4, 5, 100)[:, ::2]):
        q, s = quantize_rows_int8(x)
        rq, rs = R.quantize(x)
        assert q.shape == x.shape and s.shape == x.shape[:-1]
        assert torch.equal(q.double(), rq) and torch.equal(s.double(), rs)
    q, s = quantize_rows_int8(base[:0])
    assert q.shape == (0, 100) and s.shape == (0,)


# ---- one linear ------------------------------------------------------------------------------------------
SIZES = [(1, 1, 1), (1, 16, 16), (3, 40, 7), (17, 33, 50), (1, 2048, 512), (5, 128, 2048), (16, 4096, 256), (31, 256, 144),
         (64, 112, 272), (130, 768, 528), (257, 1040, 256), (500, 384, 1000), (513, 144, 768), (2050, 256, 320)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear(dtype, M, K, N):
    g = gen(M + K + N)
    x = hidden(g, M, K, dtype=dtype)
    w, s = weight(g, N, K)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = w8a8_gemm(x, w, s, status=status)
    q, sx = R.quantize(x)
    assert out.dtype == dtype and status.item() == 0
    R.assert_close(out, R.product(q, sx, w, s))
    same = w8a8_gemm(q.to(torch.int8), w, s, x_scale=sx.float(), out_dtype=dtype)
    assert torch.equal(out, same)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1, 16, 1), (2, 512, 48), (3, 272, 17), (4, 4096, 100), (7, 2064, 31), (8, 4096, 33),
                                   (9, 2048, 272), (16, 2048, 1000), (16, 16, 16), (1, 32768, 20), (13, 2512, 5)])
def test_linear_of_a_few_rows(dtype, M, K, N):
    """One launch that quantises the rows itself: the same numbers as from rows quantised before."""
    g = gen(M * K + N)
    x = hidden(g, M, K + 16, dtype=dtype)[:, :K]                 # rows that lie apart
    w, s = weight(g, N, K)
    out = w8a8_gemm(x, w, s)
    q, sx = R.quantize(x)
    R.assert_close(out, R.product(q, sx, w, s))
    assert torch.equal(out, w8a8_gemm(q.to(torch.int8), w, s, x_scale=sx.float(), out_dtype=dtype))
    for out_dtype in DTYPES:
        R.assert_close(w8a8_gemm(x, w, s, out_dtype=out_dtype), R.product(q, sx, w, s))
    x = x.clone()
    x[M // 2, K // 3] = float("nan")
    x[0, K - 1] = float("inf")
    bad = w8a8_gemm(x, w, s)
    assert torch.isnan(bad[M // 2]).all() and torch.isnan(bad[0]).all()
    keep = [m for m in range(M) if m not in (0, M // 2)]
    assert torch.equal(bad[keep], out[keep])


@pytest.mark.parametrize("M", [1, 40, 300])
def test_linear_sums_are_exact_at_the_largest_magnitudes(M):
    """All products 128 * 128: the int32 sum reaches 2^31 - 2^14 at the longest K."""
    K = 131071
    x = torch.full((M, K), -128, dtype=torch.int8, device=DEV)
    w = torch.full((8, K), -128, dtype=torch.int8, device=DEV)
    w[1] = 127
    ones = torch.ones(M, device=DEV), torch.ones(8, device=DEV)
    out = w8a8_gemm(x, w, ones[1], x_scale=ones[0], out_dtype=torch.float32)
    R.assert_close(out, x.double() @ w.double().T)


def test_linear_rows_without_numbers_stay_their_own():
    g = gen(5)
    x = hidden(g, 70, 256)
    x[0, 0], x[33, 7], x[69] = float("inf"), float("nan"), 0
    w, s = weight(g, 144, 256)
    out = w8a8_gemm(x, w, s)
    q, sx = R.quantize(x)
    R.assert_close(out, R.product(q, sx, w, s))
    assert torch.isnan(out[0]).all() and torch.isnan(out[33]).all() and not out[69].any()
    assert not torch.isnan(out[1:33]).any()


def test_linear_operands_off_the_grid_and_views():
    g = gen(6)
    w, s = weight(g, 144, 256)
    raw = torch.empty(144 * 256 + 1, dtype=torch.int8, device=DEV)
    raw[1:] = w.flatten()
    x = hidden(g, 50, 300)[:, 20:276]
    ref = w8a8_gemm(x.contiguous(), w, s)
    assert torch.equal(w8a8_gemm(x, raw[1:].view(144, 256), s), ref)
    assert torch.equal(w8a8_gemm(x, w.t().contiguous().t(), s.repeat_interleave(2)[::2]), ref)
    assert w8a8_gemm(x[:0], w, s).shape == (0, 144)


def test_linear_module():
    g = gen(7)
    lin = torch.nn.Linear(256, 144, bias=False).to(DEV)
    layer = LinearW8A8.from_float(lin)
    x = hidden(g, 2, 3, 256, dtype=torch.float16)
    out = layer(x)
    assert out.shape == (2, 3, 144) and out.dtype == torch.float16
    q, sx = R.quantize(x)
    R.assert_close(out, R.product(q, sx, layer.qweight, layer.scales))
    # against the float layer: half a quantisation step of each factor, K products
    full = x.double() @ lin.weight.double().T
    step = (sx[..., None] * lin.weight.double().abs().sum(1) + layer.scales.double() * x.double().abs().sum(-1, keepdim=True)) / 2
    assert ((out.double() - full).abs() <= step * 1.02 + full.abs() * 2.0 ** -10).all()
    layer.check_status()


# ---- experts ---------------------------------------------------------------------------------------------
COUNTS = [[0, 0, 3, 0], [1], [1, 0, 31, 32, 33], [128, 129, 0, 256, 257, 1], [512, 513, 545, 2, 1025], [3] * 70,
          [20] * 20 + [1100] + [300, 20] + [7, 0, 31] * 16]
WIDTHS = [(256, 128), (144, 272), (768, 384), (100, 50)]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{max(c)}")
@pytest.mark.parametrize("K,N", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_experts(counts, K, N, dtype):
    E, S = len(counts), sum(counts)
    g = gen(S + K)
    x = hidden(g, S, K, dtype=dtype)
    w, s = weight(g, E, N, K)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = w8a8_grouped_gemm(x, w, s, offsets(counts), status=status)
    h = w8a8_grouped_swiglu(x, w, s * 0.05, offsets(counts, torch.int64), status=status)
    perm = torch.randperm(S, generator=g, device=DEV).to(torch.int32)
    back = torch.empty_like(x)
    back[perm.long()] = x
    gathered = w8a8_grouped_swiglu_gather(back, perm, 1, w, s * 0.05, offsets(counts), status=status)
    assert status.item() == 0
    assert torch.equal(gathered, h)
    q, sx = R.quantize(x)
    lo = 0
    for e, n in enumerate(counts):
        rows = slice(lo, lo + n)
        R.assert_close(out[rows], R.product(q[rows], sx[rows], w[e], s[e]))
        ref, size = R.swiglu(q[rows], sx[rows], w[e], s[e] * 0.05)
        R.assert_close(h[rows], ref, R.swiglu_extra(size))
        lo += n


def test_experts_of_a_routing():
    """top_k slots of a token read one quantised row."""
    T, K, E, H, I = 90, 4, 16, 256, 128
    g = gen(11)
    x = hidden(g, T, H)
    ids = torch.rand(T, E, generator=g, device=DEV).topk(K, dim=1).indices
    perm, inv, off32, _ = moe_permute_plan(ids.to(torch.int32), E, want_int64_offsets=False)
    w, s = weight(g, E, 2 * I, H)
    s = s * 0.05
    h = w8a8_grouped_swiglu_gather(x, perm, K, w, s, off32)
    assert torch.equal(h, w8a8_grouped_swiglu(x[perm.long() // K], w, s, off32))
    q, sx = quantize_rows_int8(x)
    assert torch.equal(h, w8a8_grouped_swiglu_gather(q, perm, K, w, s, off32, x_scale=sx, out_dtype=torch.bfloat16))


@pytest.mark.parametrize("K,N", [(128, 256), (52, 30)])
def test_rows_outside_the_groups(K, N):
    g = gen(12)
    x = hidden(g, 300, K)
    w, s = weight(g, 3, N, K)
    off = torch.tensor([10, 40, 40, 290], dtype=torch.int32, device=DEV)
    out = w8a8_grouped_gemm(x, w, s, off)
    assert not out[:10].any() and not out[290:].any() and out[10:290].any()
    kept = torch.full((300, N), 7.0, dtype=torch.bfloat16, device=DEV)
    got = w8a8_grouped_gemm(x, w, s, off, out=kept)
    assert got is kept and (kept[:10] == 7).all() and (kept[290:] == 7).all() and torch.equal(kept[10:290], out[10:290])
    h = w8a8_grouped_swiglu(x, w, s, off)
    assert not h[:10].any() and not h[290:].any()
    # group g of G * E on expert g % E
    twice = torch.tensor([0, 5, 9, 20, 30, 30, 50], dtype=torch.int32, device=DEV)
    out = w8a8_grouped_gemm(x[:50], w, s, twice)
    six = w8a8_grouped_gemm(x[:50], w.repeat(2, 1, 1), s.repeat(2, 1), twice)
    assert torch.equal(out, six)


def test_offsets_and_rows_outside_x_are_not_addresses():
    """A caller's mistake stays inside the tensors: offsets past S end at S, permutation entries past x read its last row."""
    g = gen(13)
    x = hidden(g, 40, 128)
    w, s = weight(g, 2, 256, 128)
    off = torch.tensor([-3, 20, 400], dtype=torch.int32, device=DEV)
    out = w8a8_grouped_gemm(x, w, s, off)
    assert torch.equal(out, w8a8_grouped_gemm(x, w, s, offsets([20, 20])))
    assert w8a8_grouped_gemm(x, w, s, torch.zeros(3, dtype=torch.int32, device=DEV)).count_nonzero() == 0


def test_calls_on_two_streams_and_replayed():
    g = gen(14)
    x = hidden(g, 120, 256)
    w, s = weight(g, 4, 256, 256)
    off = offsets([30, 0, 50, 40])
    ref = w8a8_grouped_swiglu(x, w, s * 0.05, off), w8a8_gemm(x, w[0], s[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs.append([(w8a8_grouped_swiglu(x, w, s * 0.05, off), w8a8_gemm(x, w[0], s[0])) for _ in range(5)])
    torch.cuda.synchronize()
    for a, b in outs[0] + outs[1]:
        assert torch.equal(a, ref[0]) and torch.equal(b, ref[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = w8a8_grouped_swiglu(x, w, s * 0.05, off), w8a8_gemm(x, w[0], s[0])
    for _ in range(3):
        x.copy_(x * 0.5)                                         # scales halve, q stays
        graph.replay()
        assert torch.equal(got[1], w8a8_gemm(x, w[0], s[0])) and torch.equal(got[0], w8a8_grouped_swiglu(x, w, s * 0.05, off))


def test_refusals():
    x, w, s = torch.zeros(4, 32, device=DEV), torch.zeros(3, 16, 32, dtype=torch.int8, device=DEV), torch.zeros(3, 16, device=DEV)
    off = offsets([1, 1, 2])
    bad = [lambda: w8a8_gemm(x[:, :31], w[0], s[0]), lambda: w8a8_gemm(x, w[0].float(), s[0]),
           lambda: w8a8_gemm(x, w[0], s[0].half()), lambda: w8a8_gemm(x, w[0], s[0, :15]),
           lambda: w8a8_gemm(x.to(torch.int8), w[0], s[0]), lambda: w8a8_gemm(x, w[0], s[0], x_scale=torch.ones(4, device=DEV)),
           lambda: w8a8_gemm(x, w[0], s[0], out_dtype=torch.int32), lambda: w8a8_gemm(x.double(), w[0], s[0]),
           lambda: w8a8_gemm(x, w, s), lambda: w8a8_gemm(x, w[0].cpu(), s[0]),
           lambda: w8a8_grouped_gemm(x, w, s, offsets([1, 3])), lambda: w8a8_grouped_gemm(x, w, s, off.float()),
           lambda: w8a8_grouped_gemm(x, w, s, off, out=torch.zeros(4, 15, device=DEV)),
           lambda: w8a8_grouped_swiglu(x, w[:, :15], s[:, :15], off),
           lambda: w8a8_grouped_swiglu_gather(x, torch.zeros(4, dtype=torch.int64, device=DEV), 1, w, s, off),
           lambda: w8a8_grouped_swiglu_gather(x, torch.zeros(4, dtype=torch.int32, device=DEV), 0, w, s, off),
           lambda: w8a8_grouped_swiglu_gather(x[:0], torch.zeros(4, dtype=torch.int32, device=DEV), 1, w, s, off),
           lambda: quantize_rows_int8(x.to(torch.int32)), lambda: quantize_rows_int8(x[:, :0]),
           lambda: w8a8_gemm(torch.zeros(1, 131072, device=DEV), torch.zeros(1, 131072, dtype=torch.int8, device=DEV),
                             torch.ones(1, device=DEV))]
    for call in bad:
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -110, 2.0 ** 100])
def test_values_at_and_beside_every_half(dtype, size):
    """The numbers nearest to (n + 1/2) * scale and their neighbours, for every n and many scales: the nearest whole number of
    the exact quotient, halves to even."""
    if dtype == torch.float16:
        size = 1.0 if size < 1 else 2.0 ** 8
    g = torch.Generator().manual_seed(11)
    top = torch.cat([torch.tensor([1.0, 1.5, 127.0, 254.0 / 256, 1.0 + 2.0 ** -7]), 1 + torch.rand(59, generator=g)]) * size
    top = top.to(dtype)
    scale = R.quantize(top[:, None])[1].double()                                     # of a row that holds only its maximum
    half = (torch.arange(-127, 127).double() + 0.5) * scale[:, None]
    near = half.to(dtype)
    bits = {4: torch.int32, 2: torch.int16}[near.element_size()]
    beside = [(near.view(bits) + i).view(dtype) for i in (-2, -1, 0, 1, 2)]          # neighbours in magnitude
    x = torch.cat([top[:, None], *beside], 1)
    x = torch.where(x.abs() > top[:, None].abs(), top[:, None], x)
    x = torch.cat([x, torch.zeros(x.shape[0], -x.shape[1] % 8, dtype=dtype)], 1)
    rq, rs = R.quantize(x)
    for data in (x, torch.cat([x, x], 1)[:, 1:x.shape[1] + 1]):                      # whole vectors, and rows off their grid
        q, s = quantize_rows_int8(data.to(DEV))
        want = rq if data is x else torch.cat([rq, rq], 1)[:, 1:x.shape[1] + 1]
        assert torch.equal(s.cpu().double(), rs) and torch.equal(q.cpu().double(), want)


@pytest.mark.parametrize("rows,cols", [(4096, 1032), (4097, 2048), (4099, 4096), (4101, 2056), (5001, 1024), (4098, 768)])
def test_many_rows(rows, cols):
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, cols, generator=g).bfloat16()
    x[rows - 1, 0] = float("nan")
    x[rows // 2] = 0
    q, s = quantize_rows_int8(x.to(DEV))
    rq, rs = R.quantize(x)
    assert torch.equal(q.cpu().double(), rq)
    assert torch.equal(torch.nan_to_num(s.cpu().double(), nan=-1.0), torch.nan_to_num(rs, nan=-1.0))
