"""Rows of 8-bit codes: the quantisation, the norm that ends in it and the matrix product, each against a statement of its formula in 64 bits.

The codes are whole numbers defined without a rounding, so they are compared for equality: in float64 the quotient ``127 y / max |y|`` of two float32
numbers is formed to 2^-53, and a quotient that is not a half is at least 2^-34 of itself away from one (``254 y`` and ``(2 n + 1) max |y|`` have at most 32
significant bits).  Sums of products are compared through what was made of them: integers below 2^53 are exact in float64."""
import pytest
import torch

from spyinfer_b200 import kernels
from spyinfer_b200.kernels import Int8Rows, KernelError

DEV = "cuda:0"
gpu = pytest.mark.gpu
STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}      # a rounding is off by at most this, relative to the value


@pytest.fixture(autouse=True)
def guard_zones(guarded_allocations, monkeypatch):
    """Tensors made by strides lie between guard zones as well; the zone behind a matrix of codes begins where its last row ends."""
    plain = torch.empty_strided

    def empty_strided(size, stride, **kwargs):
        if guarded_allocations._plain(kwargs):
            return plain(size, stride, **kwargs)
        extent = 1 + sum((n - 1) * s for n, s in zip(size, stride)) if all(size) else 0
        return torch.empty((extent,), **kwargs).as_strided(size, stride)

    monkeypatch.setattr(torch, "empty_strided", empty_strided)
    yield guarded_allocations


def codes_of(y):
    """(codes, largest size, usable) of float32 rows, in 64 bits."""
    y = y.double()
    top = y.abs().amax(1) if y.shape[1] else y.new_zeros(y.shape[0])
    fine = torch.isfinite(y).all(1)
    safe = torch.where(fine & (top > 0), top, torch.ones_like(top))
    q = torch.round(torch.where(fine[:, None], y, torch.zeros_like(y)) * 127.0 / safe[:, None])
    return q.to(torch.int64), top, fine


def check_rows(got, y, factor=None, factor_err=0.0):
    """The codes of float32 rows ``y`` exactly; the scales to their roundings (one division, one product) and what ``factor`` is off by."""
    q, top, fine = codes_of(y)
    assert torch.equal(got.codes.to(torch.int64), q)
    want = top / 127.0 * (1.0 if factor is None else factor)
    err = (got.scales.double() - want).abs()
    assert bool((err[fine] <= (2.1 * 2.0 ** -24 + factor_err) * want[fine] + 2.0 ** -149).all())
    assert bool(torch.isnan(got.scales[~fine]).all())


def wild_rows(rows, length, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(rows, length, generator=g, device=DEV) * torch.exp(2.0 * torch.randn(rows, length, generator=g, device=DEV))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("length", [1, 2, 7, 8, 15, 16, 33, 100, 513, 1000, 4096, 4999, 8200, 12288, 16392, 20001, 32768, 32769, 40008])
@pytest.mark.parametrize("rows", [1, 5, 530])
def test_quantize(rows, length, dtype):
    x = wild_rows(rows, length).to(dtype)
    check_rows(kernels.quantize_int8(x), x.float())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("length", [40, 257, 4096, 16400, 33000])
def test_quantize_rows_at_the_edges(length, dtype):
    """Halves between two codes in both directions, the smallest and largest numbers, zeros of both signs, and rows that are not finite beside
    rows that are."""
    top = torch.finfo(dtype).max
    tiny = 2.0 ** -149 if dtype == torch.float32 else 2.0 ** -133
    x = wild_rows(12, length, 3)
    x[0] = (torch.arange(length, device=DEV) % 254 - 127).float() + 0.5      # halves, with the largest size 127
    x[0, 0] = 127.0
    x[1] = 0.0
    x[2] = -0.0
    x[3] = x[0] * 2.0 ** -120
    x[4] = torch.where(x[4] > 0, tiny, -3 * tiny)
    x[5] = 0.0
    x[5, length // 2] = tiny
    x[6] = torch.where(x[6] > 1.0, top, x[6].clamp(-1.0, 1.0) * 1e36)
    x[6, 3] = -top
    x[7, length - 1] = float("nan")
    x[8, 0] = float("inf")
    x[9, length // 3], x[9, length // 2] = float("-inf"), float("nan")
    x[10] = x[0] * 2.0 ** 117
    x = x.to(dtype)
    got = kernels.quantize_int8(x)
    check_rows(got, x.float())
    assert float(got.scales[1]) == 0.0 and int(got.codes[7:10].abs().max()) == 0
    assert int(got.codes.min()) >= -127


@gpu
@pytest.mark.parametrize("rows,length", [(1024, 64), (1100, 8208), (4200, 4096), (16500, 1024), (1030, 16392), (1025, 32768), (1300, 1003)])
def test_quantize_many_rows(rows, length):
    """The shares of a row that many rows are given, at their limits."""
    for dtype in (torch.bfloat16, torch.float32):
        x = wild_rows(rows, length, 9).to(dtype)
        x[rows - 1, length - 1] = float("inf")
        x[rows - 2] = 0.0
        check_rows(kernels.quantize_int8(x), x.float())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_views(dtype):
    """Rows that lie apart or start off a 16-byte border, and codes into a part of a wider matrix, whose other bytes stay."""
    wide = wild_rows(40, 300, 5).to(dtype)
    for first, end in ((0, 128), (8, 264), (1, 258), (3, 4)):
        check_rows(kernels.quantize_int8(wide[:, first:end]), wide[:, first:end].float())
    held = torch.full((42, 320), 77, dtype=torch.int8, device=DEV)
    scales = torch.full((42,), 9.0, device=DEV)
    out = Int8Rows(held[1:41, 16:16 + 250], scales[1:41])
    kernels.quantize_int8(wide[:, :250], out)
    check_rows(out, wide[:, :250].float())
    held[1:41, 16:16 + 250] = 77
    assert bool((held == 77).all()) and float(scales[0]) == float(scales[41]) == 9.0


@gpu
@pytest.mark.parametrize("xd,dd,wd", [(torch.float32, torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32, torch.bfloat16),
                                      (torch.float32, torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16, torch.float32),
                                      (torch.bfloat16, torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("rows,length", [(1, 1), (3, 8), (2, 100), (4, 1001), (1, 4096), (520, 64), (515, 4096), (3, 5120), (2, 8200), (513, 8200), (2, 16392),
                                         (2, 32768), (3, 20003)])
def test_norm(rows, length, xd, dd, wd):
    """The stream after the sum, the codes and the scales: alone, with a delta, with a stack of partial sums, and gathered.  The mean square is a
    sum of positive terms: any order of summation is off by at most (terms + 2) roundings, the inverse root by half of that and two more."""
    x, w = wild_rows(rows, length, 1).to(xd), (1 + 0.2 * torch.randn(length, device=DEV)).to(wd)
    delta, stack, eps = wild_rows(rows, length, 2).to(dd), wild_rows(3 * rows, length, 4).view(3, rows, length), 1e-5

    def check(got, v):
        factor = 1.0 / torch.sqrt(v.double().square().mean(1) + eps)
        check_rows(got, v * w.float(), factor, (length / 2 + 4) * 2.0 ** -24)

    check(kernels.rmsnorm_int8(x, w, eps), x.float())
    total = x.float() + delta.float()
    kept = x.clone()
    check(kernels.rmsnorm_int8(x, w, eps, delta=delta), total)
    assert torch.equal(x, kept)
    check(kernels.rmsnorm_int8(x, w, eps, delta=delta, write_back=True), total)
    assert torch.equal(x, total.to(xd))
    x = kept.clone()
    total = ((x.float() + stack[0]) + stack[1]) + stack[2]
    check(kernels.rmsnorm_int8(x, w, eps, delta=stack, write_back=True), total)
    assert torch.equal(x, total.to(xd))
    picked = torch.tensor([rows - 1, 0, rows // 2, 0], dtype=torch.int32, device=DEV)
    check(kernels.rmsnorm_int8(kept, w, eps, delta=delta, rows=picked), (kept.float() + delta.float())[picked.long()])


@gpu
def test_norm_rows_at_the_edges():
    length, eps = 72, 1e-6
    x = wild_rows(6, length, 7)
    w = 1 + 0.2 * torch.randn(length, device=DEV)
    x[0] = 0.0
    x[1, 5] = float("nan")
    x[2, 71] = float("inf")
    x[3] *= 2.0 ** -126
    x[4] *= 2.0 ** -30
    got = kernels.rmsnorm_int8(x, w, eps)
    check_rows(got, x * w, 1.0 / torch.sqrt(x.double().square().mean(1) + eps), (length / 2 + 4) * 2.0 ** -24)
    assert float(got.scales[0]) == 0.0 and bool(torch.isnan(got.scales[1:3]).all()) and bool(torch.isfinite(got.scales[3:]).all())


def rows_of_codes(rows, length, seed, pitch=None, full=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    pitch = pitch or (length + 15) // 16 * 16
    held = torch.full((rows, pitch), -99, dtype=torch.int8, device=DEV)       # what lies between the rows must not count
    held[:, :length] = torch.randint(-128, 128, (rows, length), generator=g, device=DEV, dtype=torch.int64).to(torch.int8) if not full else full
    return Int8Rows(held[:, :length], 0.01 * torch.rand(rows, generator=g, device=DEV) + 1e-4)


def product_of(a, w):
    """The product in 64 bits: the sums are whole numbers below 2^53."""
    return (a.codes.double() @ w.codes.double().t()) * a.scales.double()[:, None] * w.scales.double()


def check_product(got, ref, dtype):
    assert got.dtype == dtype
    err = (got.double() - ref).abs()
    # the sum to 32 bits, two products, and the result's own rounding
    assert bool((err <= (STEP[dtype] + 3.1 * 2.0 ** -24) * ref.abs()).all()), float((err / ref.abs().clamp_min(1e-300)).max())


def check_gated(got, ref, ref_err=0.0):
    g, u = ref[:, 0::2], ref[:, 1::2]
    want = g * torch.sigmoid(g) * u
    # beside the result's rounding: gate and up to 3 roundings each (the gate's also through the exponential), an exponential to 2 + |g| steps of
    # 2^-22, a division and a product
    tol = (2.0 ** -8 + (8 + 2 * g.abs()) * 2.0 ** -22) * want.abs() + 1e-37 * u.abs()
    err = (got.double() - want).abs()
    assert got.dtype == torch.bfloat16 and bool((err <= tol).all()), float((err / tol).max())


SHAPES = [(1, 1, 1), (1, 33, 16), (2, 130, 15), (3, 64, 127), (7, 4, 128), (16, 200, 129), (17, 256, 700), (32, 129, 144), (33, 1000, 300), (64, 132, 2055),
          (65, 300, 4100), (100, 4100, 512), (128, 514, 1024), (129, 5003, 257), (200, 260, 640), (256, 9600, 130), (257, 1187, 384), (301, 5003, 96),
          (520, 4864, 320), (1031, 2570, 160), (2050, 1030, 64), (700, 70, 1000)]


@gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(M, N, K):
    a, w = rows_of_codes(M, K, 1), rows_of_codes(N, K, 2)
    ref = product_of(a, w)
    for dtype in (torch.bfloat16, torch.float32):
        got = kernels.gemm_int8(a, w, out_dtype=dtype)
        check_product(got, ref, dtype)
        again = torch.empty(M, N, dtype=dtype, device=DEV)
        assert kernels.gemm_int8(a, w, out=again) is again and torch.equal(again, got)
    # a token's result is the same in every company
    for t in {0, M // 2, M - 1}:
        alone = kernels.gemm_int8(Int8Rows(a.codes[t:t + 1], a.scales[t:t + 1]), w, out_dtype=torch.float32)
        assert torch.equal(alone[0], got[t])


@gpu
@pytest.mark.parametrize("M,N,K", [(m, n + n % 2, k) for m, n, k in SHAPES])
def test_product_gated(M, N, K):
    a, w = rows_of_codes(M, K, 3), rows_of_codes(N, K, 4)
    w = Int8Rows(w.codes, w.scales * (8.0 / K ** 0.5))      # gates between about -30 and 30
    got = kernels.gemm_int8(a, w, epilogue="swiglu")
    check_gated(got, product_of(a, w))
    alone = kernels.gemm_int8(Int8Rows(a.codes[M - 1:], a.scales[M - 1:]), w, epilogue="swiglu")
    assert torch.equal(alone[0], got[M - 1])


# a size of each way that a product can be run, by the plan of 148 SMs: tokens a block 16, 32, 64, 128; K whole, cut 2, 4, 8 ways; tiles of 64, 96, 128 weight
# rows; pairs of blocks with one to five token tiles, even and uneven
# (by the plan as it is now these reach pairs with 1, 2, 3, 4, 6 and 9 token tiles of 96, 160 and 192 tokens, and single blocks but for 128 tokens by 64 weight rows;
# MORE_WAYS below has the rest, and test_sizes_reach_every_plan fails when a change of the plan leaves a way without a size)
EVERY_WAY = [(72, 14486, 306), (69, 10094, 273), (65, 11354, 2020), (65, 4562, 2090), (65, 1410, 2811), (1, 1278, 271), (1, 100, 267), (1, 130, 517), (1, 132, 1093),
             (1, 130, 2062), (19, 15348, 262), (18, 15804, 1105), (38, 100, 258), (17, 4972, 1021), (39, 142, 1065), (35, 132, 2246), (33, 14772, 278), (66, 66, 296),
             (65, 4546, 268), (35, 8786, 2069), (71, 140, 1413), (72, 130, 2414), (139, 29266, 532), (185, 27562, 651), (260, 22444, 709), (739, 8604, 795),
             (846, 1354, 4280), (258, 16242, 783), (402, 12298, 795), (324, 3958, 3491), (903, 2614, 2055)]


@gpu
@pytest.mark.parametrize("M,N,K", EVERY_WAY)
def test_product_in_every_way(M, N, K):
    """Results that leave one by one (N no multiple of 8) and in rows of 16 bytes (N a multiple of 16)."""
    for n in (N, N + -N % 16):
        a, w = rows_of_codes(M, K, 5), rows_of_codes(n, K, 6)
        w = Int8Rows(w.codes, w.scales * (8.0 / K ** 0.5))
        ref = product_of(a, w)
        for dtype in (torch.bfloat16, torch.float32):
            check_product(kernels.gemm_int8(a, w, out_dtype=dtype), ref, dtype)
        check_gated(kernels.gemm_int8(a, w, epilogue="swiglu", w_settled=True), ref)


@gpu
@pytest.mark.parametrize("M", [3, 140])
def test_product_of_the_largest_sums(M):
    """K at its limit with every code -128: 2^31 - 16,384, the largest sum there is, and its negative."""
    K, N = 131071, 20000 if M > 128 else 40
    a, w = rows_of_codes(M, K, 1, full=-128), rows_of_codes(40, K, 2, full=-128)
    w.codes[5] = 127
    w = Int8Rows(w.codes[torch.arange(N, device=DEV) % 40] if N > 40 else w.codes, w.scales[torch.arange(N, device=DEV) % 40].contiguous())
    if N > 40:
        held = torch.zeros(N, (K + 15) // 16 * 16, dtype=torch.int8, device=DEV)
        held[:, :K] = w.codes
        w = Int8Rows(held[:, :K], w.scales)
    check_product(kernels.gemm_int8(a, w, out_dtype=torch.float32), product_of(a, Int8Rows(w.codes[:40], w.scales[:40])).repeat(1, N // 40), torch.float32)


@gpu
@pytest.mark.parametrize("M", [5, 150])
def test_product_scales_and_views(M):
    """Parts of wider matrices, scales of zero, and a row that is not a number: it alone gives NaN."""
    K, N = 208, 19000 if M > 128 else 131
    a, w = rows_of_codes(M, 400, 1), rows_of_codes(N, 400, 2)
    a, w = Int8Rows(a.codes[:, 32:32 + K], a.scales), Int8Rows(w.codes[:, 176:176 + K], w.scales)
    check_product(kernels.gemm_int8(a, w), product_of(a, w), torch.bfloat16)
    a.scales[1], a.scales[2], w.scales[7] = float("nan"), 0.0, 0.0
    got = kernels.gemm_int8(a, w, out_dtype=torch.float32)
    ref = product_of(a, w)
    assert bool(torch.isnan(got[1]).all()) and not bool(torch.isnan(got[torch.arange(M, device=DEV) != 1]).any())
    keep = torch.arange(M, device=DEV) != 1
    check_product(got[keep], ref[keep], torch.float32)


@gpu
@pytest.mark.parametrize("M", [1, 9, 70, 300])
def test_a_feed_forward(M):
    """Norm, gate and up with the activation, quantisation, down: each step against its formula on what the step before gave; and the whole once
    more from a captured graph, on another stream, with new inputs."""
    H, inter, eps = 320, 4736, 1e-6
    x, delta = wild_rows(M, H, 1), wild_rows(M, H, 2).to(torch.bfloat16)
    norm = (1 + 0.1 * torch.randn(H, device=DEV)).to(torch.bfloat16)
    gate_up = kernels.quantize_int8((torch.randn(2 * inter, H, device=DEV) / H ** 0.5).to(torch.bfloat16))
    down = kernels.quantize_int8((torch.randn(H, inter, device=DEV) / inter ** 0.5).to(torch.bfloat16))

    def run(stream):
        rows = kernels.rmsnorm_int8(stream, norm, eps, delta=delta, write_back=True)
        z = kernels.gemm_int8(rows, gate_up, epilogue="swiglu")
        mid = kernels.quantize_int8(z)
        return rows, z, mid, kernels.gemm_int8(mid, down)

    stream = x.clone()
    rows, z, mid, y = run(stream)
    total = x + delta.float()
    assert torch.equal(stream, total)
    check_rows(rows, total * norm.float(), 1.0 / torch.sqrt(total.double().square().mean(1) + eps), (H / 2 + 4) * 2.0 ** -24)
    check_gated(z, product_of(rows, gate_up))
    check_rows(mid, z.float())
    check_product(y, product_of(mid, down), torch.bfloat16)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        stream.copy_(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = run(stream)
        for seed in (5, 6):
            stream.copy_(wild_rows(M, H, seed))
            fresh = stream.clone()
            graph.replay()
            eager = run(fresh)
            for p, q in zip(held, eager):
                for s, t in zip(p if isinstance(p, Int8Rows) else (p,), q if isinstance(q, Int8Rows) else (q,)):
                    assert torch.equal(s, t)
            assert torch.equal(stream, fresh)
    torch.cuda.current_stream().wait_stream(side)
    assert kernels.status_word(torch.device(DEV)).tolist() == [0, 0]


@gpu
@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (40, 2048, 1024), (300, 9472, 512), (2, 40000, 256)])
def test_weights_quantised_by_the_call_ahead(M, N, K):
    """A product may follow the quantisation of its weight at once: it reads nothing of it before that has ended.  Every round has other weights in the
    same memory, so that what an earlier round left would show."""
    x = wild_rows(M, K, 1).to(torch.bfloat16)
    w = kernels.empty_int8(N, K, DEV)
    weights = [torch.randn(N, K, device=DEV).to(torch.bfloat16) * (i + 1) for i in range(4)]
    outs = []
    for i in range(12):
        kernels.quantize_int8(weights[i % 4], w)
        outs.append(kernels.gemm_int8(kernels.quantize_int8(x), w, out_dtype=torch.float32))
    for i in range(4):
        kernels.quantize_int8(weights[i], w)
        a = kernels.quantize_int8(x)
        torch.cuda.synchronize()
        check_product(outs[i], product_of(a, w), torch.float32)
        assert torch.equal(outs[i], outs[i + 4]) and torch.equal(outs[i], outs[i + 8])
        assert torch.equal(outs[i], kernels.gemm_int8(a, w, out_dtype=torch.float32, w_settled=True, prefetch=weights[0]))


@gpu
@pytest.mark.parametrize("M", [1, 300])
def test_layer_called_as_soon_as_it_is_made(M):
    """A layer's product asks for its weight ahead of the kernels before it, so the layer is there only when its weight is; also for another stream, and for
    calls one behind the other, whose kernels overlap several deep.  The memory of the weight of the layer before is handed out again."""
    from spyinfer_b200.parts.linear import Int8Linear

    a = kernels.quantize_int8(wild_rows(M, 512, 1).to(torch.bfloat16))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for i in range(4):
        weight = torch.randn(9472, 512, device=DEV) * (i + 1)
        layer = Int8Linear(weight)
        with torch.cuda.stream(side):
            outs = [layer(a, out_dtype=torch.float32)]
        outs += [layer(a, out_dtype=torch.float32) for _ in range(3)]
        torch.cuda.synchronize()
        want = product_of(a, kernels.quantize_int8(weight))
        for out in outs:
            check_product(out, want, torch.float32)
        del layer, weight


@gpu
def test_gather_of_rows_that_there_are_not():
    """An index outside the stream reads nothing: its row is not a number, the others are as they are, and the status word says so."""
    x, w = wild_rows(5, 264, 1), torch.ones(264, device=DEV)
    rows = torch.tensor([4, -1, 0, 5, 2 ** 31 - 1, 2], dtype=torch.int32, device=DEV)
    kernels.status_word(torch.device(DEV)).zero_()
    got = kernels.rmsnorm_int8(x, w, 1e-6, rows=rows)
    good = torch.tensor([0, 2, 5], device=DEV)
    want = kernels.rmsnorm_int8(x, w, 1e-6)
    assert torch.equal(got.codes[good], want.codes[torch.tensor([4, 0, 2], device=DEV)]) and torch.equal(got.scales[good], want.scales[torch.tensor([4, 0, 2], device=DEV)])
    bad = torch.tensor([1, 3, 4], device=DEV)
    assert bool(torch.isnan(got.scales[bad]).all()) and int(got.codes[bad].abs().max()) == 0
    status = kernels.status_word(torch.device(DEV))
    assert status[0].item() == 5 and status[1].item() in (1, 3, 4)
    status.zero_()


@gpu
def test_two_streams_at_once():
    """Nothing is shared between calls: products, norms and quantisations on two streams side by side give what they give alone."""
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    jobs = []
    for i, (M, N, K) in enumerate(((9, 6144, 2048), (700, 4096, 1024))):
        x, d, g = wild_rows(M, K, i), wild_rows(M, K, i + 5).to(torch.bfloat16), torch.ones(K, device=DEV)
        w = kernels.quantize_int8(torch.randn(N, K, device=DEV).to(torch.bfloat16))
        jobs.append((x, d, g, w))

    def run(job):
        x, d, g, w = job
        rows = kernels.rmsnorm_int8(x, g, 1e-6, delta=d)
        y = kernels.gemm_int8(rows, w)
        return kernels.quantize_int8(y)

    alone = [run(j) for j in jobs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[i].append(run(jobs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(r.codes, alone[i].codes) and torch.equal(r.scales, alone[i].scales) for r in got[i])


@gpu
def test_tensors_of_another_device_than_the_current_one(monkeypatch):
    """The launch goes to the current device's stream: tensors that lie elsewhere are refused."""
    a, w, x = rows_of_codes(4, 48, 1), rows_of_codes(6, 48, 2), torch.randn(4, 48, device=DEV)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call in (lambda: kernels.gemm_int8(a, w), lambda: kernels.quantize_int8(x), lambda: kernels.rmsnorm_int8(x, torch.ones(48, device=DEV), 1e-6)):
        with pytest.raises(KernelError, match="current device"):
            call()


@gpu
def test_no_rows_and_no_outputs():
    a, w = kernels.empty_int8(0, 48, DEV), rows_of_codes(20, 48, 1)
    assert tuple(kernels.gemm_int8(a, w).shape) == (0, 20)
    assert tuple(kernels.gemm_int8(w, a).shape) == (20, 0)
    assert tuple(kernels.quantize_int8(torch.empty(0, 48, device=DEV)).codes.shape) == (0, 48)
    got = kernels.rmsnorm_int8(torch.empty(0, 48, device=DEV), torch.ones(48, device=DEV), 1e-6)
    assert tuple(got.codes.shape) == (0, 48) and tuple(got.scales.shape) == (0,)


@gpu
def test_refusals():
    """What the kernels cannot index is refused on the host, with a message that says what is wrong."""
    a, w = rows_of_codes(4, 48, 1), rows_of_codes(6, 48, 2)
    x = torch.randn(4, 48, device=DEV)
    ones = torch.ones(48, device=DEV)
    odd = torch.zeros(4, 50, dtype=torch.int8, device=DEV)
    for call, message in (
            (lambda: kernels.gemm_int8(a, rows_of_codes(6, 32, 2)), "do not fit"),
            (lambda: kernels.gemm_int8(a.codes, w), "Int8Rows"),
            (lambda: kernels.gemm_int8(Int8Rows(a.codes.cpu(), a.scales.cpu()), w), "CUDA"),
            (lambda: kernels.gemm_int8(Int8Rows(a.codes.float(), a.scales), w), "int8"),
            (lambda: kernels.gemm_int8(Int8Rows(a.codes, a.scales[:3]), w), "one float32 scale"),
            (lambda: kernels.gemm_int8(Int8Rows(a.codes, a.scales.double()), w), "one float32 scale"),
            (lambda: kernels.gemm_int8(Int8Rows(a.codes, torch.ones(8, device=DEV)[::2]), w), "one float32 scale"),
            (lambda: kernels.gemm_int8(Int8Rows(odd, a.scales), rows_of_codes(6, 50, 1)), "16-byte borders"),
            (lambda: kernels.gemm_int8(Int8Rows(a.codes[:, 1:33], a.scales), rows_of_codes(6, 32, 1)), "16-byte borders"),
            (lambda: kernels.gemm_int8(Int8Rows(a.codes[:1].expand(4, 48), a.scales), w), "16-byte borders"),
            (lambda: kernels.gemm_int8(a, w, epilogue="relu"), "unknown epilogue"),
            (lambda: kernels.gemm_int8(a, rows_of_codes(5, 48, 2), epilogue="swiglu"), "even N"),
            (lambda: kernels.gemm_int8(a, w, epilogue="swiglu", out_dtype=torch.float32), "bfloat16 output"),
            (lambda: kernels.gemm_int8(a, w, out=torch.empty(4, 5, device=DEV)), "does not fit"),
            (lambda: kernels.gemm_int8(a, w, out_dtype=torch.float16), "float32 or bfloat16"),
            (lambda: kernels.gemm_int8(a, w, prefetch=x[:1].expand(4, 48)), "overlapping"),
            (lambda: kernels.gemm_int8(a, w, prefetch=x.cpu()), "prefetch lies on"),
            (lambda: kernels.gemm_int8(kernels.empty_int8(1, 131072, DEV), kernels.empty_int8(1, 131072, DEV)), "131071"),
            (lambda: kernels.gemm_int8(kernels.empty_int8(2, 0, DEV), kernels.empty_int8(2, 0, DEV)), "must lie in"),
            (lambda: kernels.quantize_int8(x.half()), "float32 or bfloat16"),
            (lambda: kernels.quantize_int8(x.cpu()), "CUDA"),
            (lambda: kernels.quantize_int8(x.t()), "rows must be contiguous"),
            (lambda: kernels.quantize_int8(x[:1].expand(4, 48)), "overlap"),
            (lambda: kernels.quantize_int8(x, kernels.empty_int8(4, 64, DEV)), "does not fit"),
            (lambda: kernels.quantize_int8(torch.empty(3, 0, device=DEV)), "must be positive"),
            (lambda: kernels.rmsnorm_int8(x, ones[:40], 1e-6), "lengths differ"),
            (lambda: kernels.rmsnorm_int8(x, ones, 1e-6, delta=x[:3]), "differs"),
            (lambda: kernels.rmsnorm_int8(x, ones, 1e-6, delta=torch.empty(0, 4, 48, device=DEV)), "empty stack"),
            (lambda: kernels.rmsnorm_int8(x, ones, 1e-6, delta=x, rows=torch.zeros(2, dtype=torch.int32, device=DEV), write_back=True), "row gather"),
            (lambda: kernels.rmsnorm_int8(x, ones, 1e-6, rows=torch.zeros(2, dtype=torch.int64, device=DEV)), "int32"),
            (lambda: kernels.rmsnorm_int8(x, ones, 1e-6, out=kernels.empty_int8(3, 48, DEV)), "expected"),
            (lambda: kernels.rmsnorm_int8(torch.empty(1, 32769, device=DEV), torch.empty(32769, device=DEV), 1e-6), "longer than 32768")):
        with pytest.raises(KernelError, match=message):
            call()


def test_rows_of_codes_start_on_borders():
    """On the CPU: the room that is made for codes, and what is refused before a device is needed."""
    for rows, length in ((1, 1), (3, 16), (4, 17), (0, 5), (5, 4096)):
        room = kernels.empty_int8(rows, length, "cpu")
        assert tuple(room.shape) == (rows, length) and room.codes.dtype == torch.int8 and room.scales.dtype == torch.float32
        assert room.codes.stride(0) % 16 == 0 and tuple(room.scales.shape) == (rows,) and room.device == torch.device("cpu")
    room = kernels.empty_int8(4, 32, "cpu")
    with pytest.raises(KernelError, match="CUDA"):
        kernels.gemm_int8(room, room)
    with pytest.raises(KernelError, match="Int8Rows"):
        kernels.gemm_int8((room.codes, room.scales), room)
    with pytest.raises(KernelError, match="CUDA"):
        kernels.quantize_int8(torch.zeros(4, 32))
    with pytest.raises(KernelError, match="CUDA"):
        kernels.rmsnorm_int8(torch.zeros(4, 32), torch.ones(32), 1e-6)


@gpu
@pytest.mark.parametrize("xd,dd", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("rows,length", [(8, 1), (8, 72), (8, 1001), (513, 1001), (8, 4096), (8, 5120), (8, 9001), (8, 12288), (8, 20003), (8, 32768)])
def test_norm_of_rows_whose_squares_exceed_32_bits(rows, length, xd, dd):
    """Finite rows of which the squares, a thread's sum of them, or only the sum over the row lie beyond the largest 32-bit number, beside ordinary rows: the
    bound of ``test_norm``, as the sum is only formed of numbers scaled by a power of two."""
    eps = 1e-6
    x, w = wild_rows(rows, length, 1), (1 + 0.1 * torch.randn(length, device=DEV).clamp(-3, 3)).to(torch.bfloat16)
    for r, size in ((0, 3e38), (1, 1e30), (2, 2e19), (3, 1.2e19), (4, 3e18), (5, 4e17)):
        x[r] = size * (0.3 + 0.4 * torch.rand(length, device=DEV)) * torch.where(torch.rand(length, device=DEV) < 0.5, 1.0, -1.0)
    x[6, length // 2] = 2e38                      # one such number among ordinary ones
    x, delta = x.to(xd), (0.01 * wild_rows(rows, length, 2)).to(dd)
    total = x.float() + delta.float()

    def check(got):
        check_rows(got, total * w.float(), 1.0 / torch.sqrt(total.double().square().mean(1) + eps), (length / 2 + 4) * 2.0 ** -24)
        assert bool((got.scales > 0).all())

    check(kernels.rmsnorm_int8(x, w, eps, delta=delta))
    check(kernels.rmsnorm_int8(x, w, eps, delta=delta, write_back=True))
    assert torch.equal(x, total.to(xd))


@gpu
@pytest.mark.parametrize("M,N,K", [(3, 400, 16), (17, 240, 2062), (70, 1410, 2811), (739, 8604, 795)])
def test_gates_far_below_zero(M, N, K):
    """The activation where its exponential leaves 32 bits or nearly does, by every way that results leave: gates from -120 to 100, closely spaced around -88,
    with ups from small to so large that the tiny activation counts."""
    gates = torch.cat([torch.linspace(-120, 100, 45), torch.linspace(-90, -85, 51), torch.tensor([0.0, -0.0, -1e-30, 1e-30, -1e30, 1e3])]).to(DEV)
    ups = torch.tensor([1.0, -3e4, 1e25, -1e33, 1e35], device=DEV)
    i = torch.arange(N // 2, device=DEV)
    held = torch.zeros(M + N, (K + 15) // 16 * 16, dtype=torch.int8, device=DEV)
    held[:M, K - 1] = 1
    scales = torch.empty(N, device=DEV)
    for first, of in ((0, gates[i % gates.numel()]), (1, ups[(i // 3) % ups.numel()])):
        held[M + first::2, K - 1] = (127 * of.sign()).to(torch.int8)
        scales[first::2] = of.abs() / 127
    a, w = Int8Rows(held[:M, :K], torch.ones(M, device=DEV)), Int8Rows(held[M:, :K], scales)
    check_gated(kernels.gemm_int8(a, w, epilogue="swiglu"), product_of(a, w))


def test_waits_for_tensor_memory_name_their_registers():
    """A load from tensor memory fills registers that may be read behind the wait only, and the pair kernel carries them over a loop's end: every wait of these
    kernels names them as read and written, so that no read can be moved ahead of it."""
    from pathlib import Path

    folder = Path(kernels.__file__).parent / "csrc"
    product, shared = (folder / "gemm_int8.cu").read_text(), (folder / "tcgen05.cuh").read_text()
    waits = [line.strip() for line in product.splitlines() if "tmem_wait_ld" in line]
    assert sorted(waits) == ["tmem_wait_ld(ahead);", "tmem_wait_ld(r);", "tmem_wait_ld(r);"]
    for n in (16, 32):
        body = shared.split(f"tmem_wait_ld<{n}>", 1)[1].split("}", 1)[0]
        assert all(f'"+r"(r[{i}])' in body for i in range(n)) and "tcgen05.wait::ld" in body


# ---- nothing is read before the kernels ahead have ended ------------------------------------------------------------------------
def behind_a_product(dtype, consume, M=64, N=24576, K=4096):
    """``consume`` of what a product of some 20 us writes, launched right behind it so that its blocks start beside the product's last ones: one launch after
    the other and from a captured graph, with other inputs every time and the product's output cleared before.  What it gives has to be, to the last bit, what it
    gives of the same numbers when nothing runs any more."""
    a, w = rows_of_codes(M, K, 1), rows_of_codes(N, K, 2)
    a, w = Int8Rows(a.codes, a.scales * 0.1), w        # results near one
    z = torch.empty(M, N, dtype=dtype, device=DEV)

    def run():
        kernels.gemm_int8(a, w, out=z, w_settled=True)
        return consume(z)

    def flat(out):
        return [t for p in (out if type(out) in (tuple, list) else (out,)) for t in (p if isinstance(p, Int8Rows) else (p,))]

    run()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = run()
        for i in range(6):
            a.codes.copy_(torch.randint(-128, 128, (M, K), device=DEV).to(torch.int8))
            z.zero_()
            if i % 2:
                graph.replay()
                got = held
            else:
                got = run()
            side.synchronize()
            want = consume(z.clone())
            side.synchronize()
            for g, t in zip(flat(got), flat(want)):
                assert torch.equal(g, t) or bool(((g == t) | (torch.isnan(g) & torch.isnan(t))).all()), f"pass {i}: {int((g != t).sum())} of {g.numel()} differ"


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,length", [(64, 24576), (96, 16384), (384, 4096), (1536, 1024), (6000, 256), (300, 4999), (1100, 1001), (40, 39000)])
def test_quantisation_right_behind_what_writes_its_input(rows, length, dtype):
    behind_a_product(dtype, lambda z: kernels.quantize_int8(z.view(-1)[:rows * length].view(rows, length)))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,length", [(1, 4096), (64, 8192), (384, 4096), (1500, 1024), (300, 4999), (600, 1001), (40, 32768), (30, 20003), (80, 16392)])
def test_norm_right_behind_what_writes_its_input(rows, length, dtype):
    """The stream, the delta, the stacked delta and the weight."""
    x, weight = wild_rows(rows, length, 3), (1 + 0.1 * torch.randn(length, device=DEV)).to(torch.bfloat16)

    def norms(z):
        part = z.view(-1)[:rows * length].view(rows, length)
        half = z.view(-1)[:2 * (rows // 2) * length].view(2, rows // 2, length)
        return (kernels.rmsnorm_int8(part, weight, 1e-6), kernels.rmsnorm_int8(x, weight, 1e-6, delta=part),
                kernels.rmsnorm_int8(x[:rows // 2].contiguous(), weight, 1e-6, delta=half) if rows > 1 else kernels.rmsnorm_int8(x, weight, 1e-6))

    behind_a_product(dtype, norms)
    behind_a_product(dtype, lambda z: kernels.rmsnorm_int8(x, weight, 1e-6, delta=z.view(-1)[:rows * length].view(rows, length)))
    behind_a_product(dtype, lambda z: kernels.rmsnorm_int8(x, z.view(-1)[-length:], 1e-6))


@gpu
@pytest.mark.parametrize("M,N,K", [(1, 6144, 4096), (64, 4096, 2048), (40, 1000, 300), (300, 9472, 512), (640, 24576, 1024)])
def test_product_right_behind_what_writes_its_scales(M, N, K):
    a, w = rows_of_codes(M, K, 3), rows_of_codes(N, K, 4)
    behind_a_product(torch.float32, lambda z: kernels.gemm_int8(Int8Rows(a.codes, z.view(-1)[-M:]), w, out_dtype=torch.float32))
    behind_a_product(torch.float32, lambda z: kernels.gemm_int8(a, Int8Rows(w.codes, z.view(-1)[-N:]), out_dtype=torch.float32))
    behind_a_product(torch.float32, lambda z: kernels.gemm_int8(Int8Rows(a.codes, z.view(-1)[:M]), Int8Rows(w.codes, z.view(-1)[-N:]), epilogue="swiglu"))


# ---- which way a product is run ------------------------------------------------------------------------------------------------
SMS = 148


def way_of(M, N, K, sms=SMS):
    """Pairs: the tallest token tile, and whether others are lower.  Single blocks: tokens, ways that K is cut, and weight rows."""
    p = kernels.gemm_int8_plan(M, N, K, sms)
    return ("pairs", p.tile_tokens, (M + 31) // 32 % p.token_tiles != 0) if p.pairs else ("single", p.tile_tokens, p.k_cuts, p.tile_rows)


# what the sizes above leave out: the heights of the pairs' token tiles (64 to 256, even and uneven; from 96 on most with three or more tiles a pair, the last
# one ragged), a ring of six stages filled several times, and 128 tokens by 64 weight rows
MORE_WAYS = {(6731, 312, 434): ("single", 128, 1, 64), (368, 2836, 9251): ("pairs", 64, False), (131, 6142, 8246): ("pairs", 64, True),
             (162, 26036, 776): ("pairs", 96, False), (1283, 964, 3966): ("pairs", 96, True), (495, 13620, 977): ("pairs", 128, False),
             (477, 14008, 993): ("pairs", 128, True), (138, 50300, 280): ("pairs", 160, False), (274, 26346, 514): ("pairs", 160, True),
             (171, 55968, 286): ("pairs", 192, False), (660, 13970, 536): ("pairs", 192, True), (665, 17436, 407): ("pairs", 224, False),
             (393, 27334, 404): ("pairs", 224, True), (748, 18690, 426): ("pairs", 256, False), (907, 13986, 397): ("pairs", 256, True),
             (2041, 6150, 2200): ("pairs", 256, False), (1000, 8192, 2048): ("pairs", 256, False)}


def test_plan_of_a_product():
    """What the plan says fits the sizes, and sizes that the product refuses have none."""
    import random
    rng = random.Random(2)
    for _ in range(2000):
        M, N, K = (max(1, round(top ** rng.random())) for top in (8192, 60000, 20000))
        p = kernels.gemm_int8_plan(M, N, K, SMS)
        if p.pairs:
            runs = (M + 31) // 32
            assert p.tile_tokens % 32 == 0 and 32 <= p.tile_tokens <= 256 and p.k_cuts == 1 and p.tile_rows == 256
            assert p.tile_tokens == 32 * -(-runs // p.token_tiles) and runs >= p.token_tiles
        else:
            assert p.tile_tokens in (16, 32, 64, 128) and p.token_tiles == -(-M // p.tile_tokens) and p.tile_rows in (64, 96, 128)
            assert p.k_cuts == 1 or (p.k_cuts in (2, 4, 8) and p.tile_rows == 128 and K > 128 * (2 * p.k_cuts - 1))
    for M, N, K, sms in ((0, 1, 1, SMS), (1, 0, 1, SMS), (1, 1, 0, SMS), (1, 1, 131072, SMS), (1, 1, 1, 0), (2 ** 22 + 1, 1, 1, SMS), (1, 2 ** 40, 1, SMS)):
        with pytest.raises(KernelError, match="no plan"):
            kernels.gemm_int8_plan(M, N, K, sms)


def test_sizes_reach_every_plan():
    """The plan changes with its constants: the sizes of this file's product tests have to go every way that a product of random sizes goes."""
    import random
    for size, way in MORE_WAYS.items():
        assert way_of(*size) == way
    tested = {way_of(M, n, K) for M, N, K in SHAPES + EVERY_WAY + list(MORE_WAYS) for n in (N, N + N % 2)}
    rng = random.Random(4)
    found = set()
    for _ in range(20000):
        found.add(way_of(*(max(low, round(low * (high / low) ** rng.random())) for low, high in ((1, 8192), (1, 60000), (1, 20000)))))
    assert len(found) >= 30 and not found - tested, found - tested


@gpu
@pytest.mark.parametrize("M,N,K", list(MORE_WAYS))
def test_product_in_more_ways(M, N, K):
    """As ``test_product_in_every_way``; and a token alone, which goes another way, gives the same bits."""
    assert way_of(M, N, K, torch.cuda.get_device_properties(0).multi_processor_count) == MORE_WAYS[M, N, K]
    a, w = rows_of_codes(M, K, 5), rows_of_codes(N, K, 6)
    w = Int8Rows(w.codes, w.scales * (8.0 / K ** 0.5))
    ref = product_of(a, w)
    outs = {}
    for dtype in (torch.bfloat16, torch.float32):
        outs[dtype] = kernels.gemm_int8(a, w, out_dtype=dtype)
        check_product(outs[dtype], ref, dtype)
    gated = kernels.gemm_int8(a, w, epilogue="swiglu", w_settled=True)
    check_gated(gated, ref)
    for t in (0, 37, M // 2, M - 1):
        alone = Int8Rows(a.codes[t:t + 1], a.scales[t:t + 1])
        assert not kernels.gemm_int8_plan(1, N, K).pairs
        for dtype in outs:
            assert torch.equal(kernels.gemm_int8(alone, w, out_dtype=dtype)[0], outs[dtype][t])
        assert torch.equal(kernels.gemm_int8(alone, w, epilogue="swiglu")[0], gated[t])


# ---- what the other tests ask of a product, of products on pairs of blocks --------------------------------------------------------
@gpu
def test_pairs_scales_and_views():
    """As ``test_product_scales_and_views``."""
    M, N, K = 1000, 8192, 1024
    assert kernels.gemm_int8_plan(M, N, K).pairs
    a, w = rows_of_codes(M, 1400, 1), rows_of_codes(N, 1400, 2)
    a, w = Int8Rows(a.codes[:, 32:32 + K], a.scales), Int8Rows(w.codes[:, 176:176 + K], w.scales)
    check_product(kernels.gemm_int8(a, w), product_of(a, w), torch.bfloat16)
    a.scales[1], a.scales[2], w.scales[7] = float("nan"), 0.0, 0.0
    keep = torch.arange(M, device=DEV) != 1
    got, ref = kernels.gemm_int8(a, w, out_dtype=torch.float32), product_of(a, w)
    assert bool(torch.isnan(got[1]).all())
    check_product(got[keep], ref[keep], torch.float32)
    gated = kernels.gemm_int8(a, w, epilogue="swiglu")
    assert bool(torch.isnan(gated[1]).all())
    check_gated(gated[keep], ref[keep])


@gpu
def test_pairs_in_a_feed_forward_captured_and_replayed():
    """As ``test_a_feed_forward``: both products on pairs, run, captured on another stream and replayed with new inputs."""
    M, H, inter, eps = 1100, 2048, 5120, 1e-6
    assert kernels.gemm_int8_plan(M, 2 * inter, H).pairs and kernels.gemm_int8_plan(M, H, inter).pairs
    x, delta = wild_rows(M, H, 1), wild_rows(M, H, 2).to(torch.bfloat16)
    norm = (1 + 0.1 * torch.randn(H, device=DEV)).to(torch.bfloat16)
    gate_up = kernels.quantize_int8((torch.randn(2 * inter, H, device=DEV) / H ** 0.5).to(torch.bfloat16))
    down = kernels.quantize_int8((torch.randn(H, inter, device=DEV) / inter ** 0.5).to(torch.bfloat16))

    def run(stream):
        rows = kernels.rmsnorm_int8(stream, norm, eps, delta=delta, write_back=True)
        z = kernels.gemm_int8(rows, gate_up, epilogue="swiglu")
        mid = kernels.quantize_int8(z)
        return rows, z, mid, kernels.gemm_int8(mid, down)

    def parts(out):
        return [t for p in out for t in (p if isinstance(p, Int8Rows) else (p,))]

    stream = x.clone()
    rows, z, mid, y = run(stream)
    check_gated(z, product_of(rows, gate_up))
    check_rows(mid, z.float())
    check_product(y, product_of(mid, down), torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        stream.copy_(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = run(stream)
        for seed in (5, 6):
            stream.copy_(wild_rows(M, H, seed))
            fresh = stream.clone()
            graph.replay()
            assert all(torch.equal(s, t) for s, t in zip(parts(held), parts(run(fresh)))) and torch.equal(stream, fresh)
    torch.cuda.current_stream().wait_stream(side)
    assert kernels.status_word(torch.device(DEV)).tolist() == [0, 0]


@gpu
def test_pairs_behind_the_quantisation_of_their_weight():
    """As ``test_weights_quantised_by_the_call_ahead``."""
    M, N, K = 640, 24576, 1024
    assert kernels.gemm_int8_plan(M, N, K).pairs
    x = wild_rows(M, K, 1).to(torch.bfloat16)
    w = kernels.empty_int8(N, K, DEV)
    weights = [torch.randn(N, K, device=DEV).to(torch.bfloat16) * (i + 1) for i in range(3)]
    outs = []
    for i in range(9):
        kernels.quantize_int8(weights[i % 3], w)
        outs.append(kernels.gemm_int8(kernels.quantize_int8(x), w, out_dtype=torch.float32))
    for i in range(3):
        kernels.quantize_int8(weights[i], w)
        a = kernels.quantize_int8(x)
        torch.cuda.synchronize()
        check_product(outs[i], product_of(a, w), torch.float32)
        assert torch.equal(outs[i], outs[i + 3]) and torch.equal(outs[i], outs[i + 6])
        assert torch.equal(outs[i], kernels.gemm_int8(a, w, out_dtype=torch.float32, w_settled=True))


@gpu
def test_pairs_of_a_layer_called_as_soon_as_it_is_made():
    """As ``test_layer_called_as_soon_as_it_is_made``."""
    from spyinfer_b200.parts.linear import Int8Linear

    M, N, K = 400, 20000, 1024
    assert kernels.gemm_int8_plan(M, N, K).pairs
    a = kernels.quantize_int8(wild_rows(M, K, 1).to(torch.bfloat16))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for i in range(3):
        weight = torch.randn(N, K, device=DEV) * (i + 1)
        layer = Int8Linear(weight)
        with torch.cuda.stream(side):
            outs = [layer(a, out_dtype=torch.float32)]
        outs += [layer(a, out_dtype=torch.float32) for _ in range(3)]
        torch.cuda.synchronize()
        want = product_of(a, kernels.quantize_int8(weight))
        for out in outs:
            check_product(out, want, torch.float32)
        del layer, weight


@gpu
def test_pairs_on_two_streams_at_once():
    """As ``test_two_streams_at_once``: products on pairs on both streams."""
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    jobs = []
    for i, (M, N, K) in enumerate(((1100, 10240, 2048), (400, 20000, 1024))):
        assert kernels.gemm_int8_plan(M, N, K).pairs
        jobs.append((wild_rows(M, K, i), wild_rows(M, K, i + 5).to(torch.bfloat16), torch.ones(K, device=DEV),
                     kernels.quantize_int8(torch.randn(N, K, device=DEV).to(torch.bfloat16))))

    def run(job):
        x, d, g, w = job
        return kernels.quantize_int8(kernels.gemm_int8(kernels.rmsnorm_int8(x, g, 1e-6, delta=d), w))

    alone = [run(j) for j in jobs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[i].append(run(jobs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(r.codes, alone[i].codes) and torch.equal(r.scales, alone[i].scales) for r in got[i])
    assert kernels.status_word(torch.device(DEV)).tolist() == [0, 0]


# ---- the engine on 8-bit weights ----------------------------------------------------------------------------------------------
def plain_int8_logits(monkeypatch, weights, cfg, tokens):
    """The plain implementation with every product of the layers on quantised rows and quantised weights, in 32 bits (the sums in 64)."""
    import plain_model

    def quantised(m):
        m = m.double()
        top = m.abs().amax(1, keepdim=True).clamp_min(1e-300)
        return torch.round(m * 127.0 / top), top / 127.0

    head = weights["model.embed_tokens.weight"] if cfg.get("tie_word_embeddings", False) else weights["lm_head.weight"]
    plain = plain_model.linear

    def linear(x, w):
        if w is head:
            return plain(x, w)
        (qx, sx), (qw, sw) = quantised(x), quantised(w)
        return ((qx @ qw.t()) * sx * sw.t()).to(x.dtype)

    monkeypatch.setattr(plain_model, "linear", linear)
    try:
        return plain_model.forward_logits(weights, cfg, tokens)
    finally:
        monkeypatch.setattr(plain_model, "linear", plain)


def int8_engine(folder, **kw):
    from spyinfer_b200 import LLMEngine
    opts = dict(dtype="bfloat16", quantization="int8", max_num_seqs=4, max_model_len=256, kvcache_block_size=16, num_kvcache_blocks=64, max_num_batched_tokens=256)
    opts.update(kw)
    return LLMEngine(folder, **opts)


@gpu
@pytest.mark.parametrize("name", ["a", "b", "c", "d", "e"])
def test_engine_logits(name, tiny_models, monkeypatch):
    """A prompt whole, in portions, and its last tokens one by one, against the plain implementation on quantised weights and rows.  The engine's
    numbers between two products are rounded to bfloat16, so a few codes of a row differ by one: at most what two independent quantisations
    differ by, 0.41 of a code (rms) with the largest of a row near 2.5 times its rms, 1 % of the row; four such rows a layer in up to four
    layers add up to 4 % of the logits in the mean square if nothing damped them, and the largest of some thousand differences is to its rms
    what the largest logit is to the logits', within a factor of two."""
    from spyinfer_b200.engine.batch import StepEntry
    folder, cfg, weights = tiny_models[name]
    g = torch.Generator().manual_seed(7)
    tokens = torch.randint(0, cfg["vocab_size"], (150,), generator=g).tolist()
    want = plain_int8_logits(monkeypatch, weights, cfg, tokens).double()
    engine = int8_engine(folder)

    def check(rows, first):
        got = torch.as_tensor(rows).double()
        ref = want[first:first + got.shape[0]]
        err = (got - ref).abs()
        assert bool(torch.isfinite(got).all())
        assert float(err.max()) <= 8e-2 * float(ref.abs().max()) and float(err.square().mean().sqrt()) <= 4e-2 * float(ref.square().mean().sqrt())

    check(engine.step_raw([StepEntry("whole", tokens, list(range(150)))]), 0)
    at = 0
    for n in (7, 1, 64, 33, 40):
        check(engine.step_raw([StepEntry("parts", tokens[at:at + n], list(range(n)))]), at)
        at += n
    for at in range(145, 150):
        check(engine.step_raw([StepEntry("parts", tokens[at:at + 1], [0])]), at)
    used = {m for layer in engine.model.layers for p in layer.parts() for m in p.modules()}
    assert {"gemm_int8", "quant_int8"} <= used and not {"gemm_tcgen05", "gemm_simt", "rmsnorm"} & used


@gpu
def test_engine_generates_the_same_with_and_without_graphs(tiny_models):
    """Decode steps and small mixed steps replayed from graphs (with their hints of the next weights) against launches one by one."""
    from spyinfer_b200 import SamplingParams
    folder, cfg, _ = tiny_models["d"]
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, cfg["vocab_size"], (n,), generator=g).tolist() for n in (1, 9, 40, 130, 17, 3)]
    outs = []
    for graphs in (True, False):
        engine = int8_engine(folder, use_cuda_graphs=graphs)
        outs.append(engine.generate(prompts, SamplingParams(max_new_tokens=20, ignore_eos=True)))
        assert (engine.runner.graph_steps > 0) == graphs
        engine.runner.check_status()
    assert outs[0] == outs[1] and all(len(o) == 20 for o in outs[0])


def test_engine_options():
    from spyinfer_b200 import EngineConfig, config_from_json
    from spyinfer_b200.engine.model import Model
    from conftest import TINY
    assert EngineConfig(quantization="int8").quantization == "int8" and EngineConfig().quantization is None
    for bad in (dict(quantization="int4"), dict(quantization="int8", dtype="float32")):
        with pytest.raises(ValueError, match="quantization"):
            EngineConfig(**bad)
    spec = config_from_json(TINY["a"]["config"]).to_spec()
    model = Model(spec, torch.bfloat16, None, 256, quantization="int8")
    assert all(l.block.mixer_norm.emits_int8 and l.block.ffn_norm.emits_int8 for l in model.layers) and not model.final_norm.emits_int8
    assert not Model(spec, torch.bfloat16, None, 256).layers[0].block.mixer_norm.emits_int8
    with pytest.raises(ValueError, match="quantization"):
        Model(spec, torch.float32, None, 256, quantization="int8")


def test_other_architectures_are_refused():
    from spyinfer_b200 import config_from_json
    from spyinfer_b200.engine.model import Model
    from test_bubalix import BX
    from test_dogilorn import DG
    for config in (BX["a"]["config"], DG["a"]["config"]):
        with pytest.raises(ValueError, match="does not cover"):
            Model(config_from_json(config).to_spec(), torch.bfloat16, None, 256, quantization="int8")


def stored_as(folder, weights, cfg, dtype):
    import json
    from safetensors.torch import save_file
    folder.mkdir()
    (folder / "config.json").write_text(json.dumps(cfg))
    save_file({k: v.to(dtype).contiguous() for k, v in weights.items()}, str(folder / "model.safetensors"))
    return str(folder)


@pytest.mark.parametrize("name,stay", [("a", 1), ("b", 2)])
def test_warning_of_wide_matrices_leaves_out_what_is_quantised(name, stay, tiny_models, tmp_path, monkeypatch):
    """Of a checkpoint in 32 bits (or float16) only the table and the head stay so in a quantised model; its layers' matrices run on the tensor cores."""
    import warnings
    from spyinfer_b200 import config_from_json
    from spyinfer_b200.engine.model import Model
    _, cfg, weights = tiny_models[name]
    spec = config_from_json(cfg).to_spec()
    monkeypatch.setattr(Model, "bind", lambda self, tensors: None)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        folder = stored_as(tmp_path / str(dtype), weights, cfg, dtype)
        for quantization in (None, "int8"):
            with warnings.catch_warnings(record=True) as seen:
                warnings.simplefilter("always")
                Model(spec, torch.bfloat16, "cpu", 256, quantization=quantization).load(folder)
            if dtype == torch.bfloat16:
                assert not seen
            else:
                count = stay if quantization else stay + 7 * cfg["num_hidden_layers"]
                assert len(seen) == 1 and f": {count} matrices are stored in 32-bit" in str(seen[0].message)
                assert "embed_tokens" in str(seen[0].message)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_engine_on_a_checkpoint_in_wider_types(dtype, tiny_models, tmp_path, monkeypatch):
    """The weights are quantised from the numbers as they are stored; the bound of ``test_engine_logits``."""
    from spyinfer_b200.engine.batch import StepEntry
    _, cfg, weights = tiny_models["d"]
    weights = {k: v.float() * (1 + 2.0 ** -9) for k, v in weights.items()}          # not numbers of bfloat16
    folder = stored_as(tmp_path / "wide", weights, cfg, dtype)
    g = torch.Generator().manual_seed(9)
    tokens = torch.randint(0, cfg["vocab_size"], (90,), generator=g).tolist()
    want = plain_int8_logits(monkeypatch, {k: v.to(dtype).float() for k, v in weights.items()}, cfg, tokens).double()
    with pytest.warns(UserWarning, match="1 matrices are stored in 32-bit"):
        engine = int8_engine(folder)
    got = torch.as_tensor(engine.step_raw([StepEntry("whole", tokens, list(range(90)))])).double()
    err = (got - want).abs()
    assert bool(torch.isfinite(got).all())
    assert float(err.max()) <= 8e-2 * float(want.abs().max()) and float(err.square().mean().sqrt()) <= 4e-2 * float(want.square().mean().sqrt())
    used = {m for layer in engine.model.layers for p in layer.parts() for m in p.modules()}
    assert {"gemm_int8", "quant_int8"} <= used and not {"gemm_tcgen05", "gemm_simt"} & used


@gpu
def test_engine_steps_of_wide_layers_replayed_and_launched():
    """Layers whose products take long enough for the kernels behind them to start beside them: prompts, mixed steps and replies replayed from graphs against the
    same steps launched one by one.  Both quantise the same numbers but for what another cut of a sum makes of a rounding to bfloat16, so the bound of
    ``test_engine_logits`` holds between them; rows that were read too early would be of other tokens altogether."""
    from spyinfer_b200 import LLMEngine, config_from_json
    from spyinfer_b200.engine.batch import StepEntry
    cfg = dict(architectures=["Qwen3ForCausalLM"], model_type="qwen3", hidden_act="silu", num_hidden_layers=3, hidden_size=2048, num_attention_heads=16,
               num_key_value_heads=8, head_dim=128, intermediate_size=8192, vocab_size=4096, rope_theta=1000000.0, rms_norm_eps=1e-6,
               tie_word_embeddings=False, max_position_embeddings=4096)
    engines = [LLMEngine(model_config=config_from_json(cfg), seed=5, dtype="bfloat16", quantization="int8", use_cuda_graphs=graphs, max_num_seqs=64,
                         max_model_len=1024, kvcache_block_size=16, num_kvcache_blocks=600, max_num_batched_tokens=1024) for graphs in (True, False)]
    g = torch.Generator().manual_seed(3)

    def tokens(n):
        return torch.randint(0, 4096, (n,), generator=g).tolist()

    def step(entries):
        replayed, launched = (torch.as_tensor(e.step_raw(entries)).double() for e in engines)
        err = (replayed - launched).abs()
        assert bool(torch.isfinite(replayed).all())
        assert float(err.max()) <= 8e-2 * float(launched.abs().max()) and float(err.square().mean().sqrt()) <= 4e-2 * float(launched.square().mean().sqrt())

    for turn in range(4):
        names = [f"{turn}.{i}" for i in range(8)]
        step([StepEntry(names[0], tokens(300), [299])])
        step([StepEntry(n, tokens(k), [k - 1]) for n, k in zip(names[1:], (1, 7, 33, 64, 100, 3, 40))])
        for _ in range(5):
            step([StepEntry(n, tokens(1), [0]) for n in names])
        step([StepEntry(names[0], tokens(200), [0, 199]), StepEntry(names[1], tokens(1), [0])])
        for e in engines:
            for n in names:
                e.runner.finish(n)
    assert engines[0].runner.graph_steps > 20 and engines[1].runner.graph_steps == 0
    for e in engines:
        e.runner.check_status()
