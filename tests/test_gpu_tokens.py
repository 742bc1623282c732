"""GPU: quantise / dequantise per token and the 8-bit product with parameters per token and channel, against the oracle row by
row and an integer reference whose float steps are made one by one (so the comparison is for equal bits)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]


def rows_of(torch, seed, M, K, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))
    if M > 2:
        x[1] = x[1].abs()          # a row that does not straddle zero, and its mirror image
        x[2] = -x[2].abs()
    return x.to(getattr(torch, dtype))


def oracle_rows(oracle, x):
    """codes, scale, zero point of every row by the per-tensor functions of the oracle."""
    P = oracle.port
    codes, scales, zeros = [], [], []
    for row in x.float().numpy():
        row = np.ascontiguousarray(row)
        lo, hi = P.get_min_max(row)
        qp = P.compute_qparams(lo, hi)
        codes.append(P.quantize_u8(row, qp))
        scales.append(np.float32(qp.scale))
        zeros.append(int(qp.zero_point))
    return np.stack(codes), np.array(scales, np.float32), np.array(zeros, np.uint8)


def unpack(qparams):
    raw = qparams.cpu().numpy()
    return raw.view(np.float32)[:, 0].copy(), raw[:, 4].copy()


def values_f32(codes, scale, zero):
    return scale[:, None] * (codes.astype(np.float32) - zero[:, None].astype(np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 2), (1, 7), (5, 8), (9, 100), (4, 128), (33, 512), (3, 1000), (7, 1021), (2, 1024), (3, 1032),
                                 (5, 2047), (4, 2048), (3, 4096), (1, 4104), (2, 8192), (3, 12000), (2, 16384), (2, 16400), (2, 20001), (1500, 64)])
def test_quantize_tokens_equals_the_per_tensor_functions_row_by_row(cuda, oracle, dtype, M, K):
    import ltq
    x = rows_of(cuda, 1000 * M + K, M, K, dtype)
    q, qp, sums = ltq.quantize_tokens(x.cuda())
    codes, scales, zeros = oracle_rows(oracle, x)
    s, z = unpack(qp)
    assert np.array_equal(s, scales) and np.array_equal(z, zeros)
    assert np.array_equal(q.cpu().numpy(), codes)
    assert np.array_equal(sums.cpu().numpy(), codes.astype(np.int64).sum(1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [96, 97, 3000, 20001])
def test_rows_that_the_per_tensor_functions_leave_undefined(cuda, oracle, dtype, K):
    """Zeros, subnormal ranges, ranges that overflow, infinities and NaN; their neighbours are not touched."""
    import ltq
    torch = cuda
    x = rows_of(torch, 5, 12, K, dtype).float()
    tiny = {"float32": 1e-42, "float16": 6e-8, "bfloat16": 1e-39}[dtype]
    big = torch.finfo(getattr(torch, dtype)).max
    x[0] = 0
    x[2] = 0
    x[2, K // 2] = tiny
    x[4, 0], x[4, 1] = big, -big
    x[6, K - 1] = float("inf")
    x[8, 3] = float("-inf")
    x[10, K // 3] = float("nan")
    x[11, 0], x[11, 1] = float("inf"), float("nan")
    x = x.to(getattr(torch, dtype))
    q, qp, sums = ltq.quantize_tokens(x.cuda())
    q, (s, z), sums = q.cpu().numpy(), unpack(qp), sums.cpu().numpy()
    normal = [1, 3, 5, 7, 9]
    codes, scales, zeros = oracle_rows(oracle, x[normal])
    assert np.array_equal(q[normal], codes) and np.array_equal(s[normal], scales) and np.array_equal(z[normal], zeros)
    assert s[0] == np.float32(2.0 ** -126) and z[0] == 0 and not q[0].any() and sums[0] == 0
    xf = x.float().numpy()
    floor = np.float32(2.0 ** -126)
    want = max(np.float32(xf[2].max() / np.float32(255)), floor)
    assert s[2] == want and z[2] == 0
    assert q[2].max() == int(np.floor(np.float64(np.float32(xf[2].max() / want)) + 0.5))
    lo, hi = np.float32(xf[4].min()), np.float32(xf[4].max())
    if dtype == "float16":
        want = np.float32((hi - lo) / np.float32(255))
    else:
        with np.errstate(over="ignore"):
            assert np.isinf(hi - lo)
        want = np.float32(hi / np.float32(255)) - np.float32(lo / np.float32(255))
    # zero point round(127.5 give or take a rounding), codes by the rule's own float steps
    assert s[4] == want and z[4] == int(np.floor(np.float64(np.float32(0) - np.float32(lo / want)) + 0.5))
    v = np.clip((np.float32(z[4]) + (xf[4] / want).astype(np.float32)).astype(np.float32), 0, 255)
    assert np.array_equal(q[4], np.floor(v.astype(np.float64) + 0.5).astype(np.uint8))
    for r in (6, 8, 10, 11):
        assert np.isnan(s[r]) and z[r] == 0 and not q[r].any() and sums[r] == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,ld,first", [(256, 300, 0), (256, 264, 8), (255, 256, 0), (64, 64 + 3, 1), (4096, 5000, 4)])
def test_strided_rows(cuda, oracle, dtype, K, ld, first):
    import ltq
    buf = rows_of(cuda, 7, 6, ld, dtype)
    x = buf[:, first:first + K]
    dev = buf.cuda()
    q, qp, sums = ltq.quantize_tokens(dev[:, first:first + K])
    codes, scales, zeros = oracle_rows(oracle, x)
    assert np.array_equal(q.cpu().numpy(), codes) and np.array_equal(unpack(qp)[0], scales)
    out = cuda.full((6, ld), 7.0, dtype=getattr(cuda, dtype), device="cuda")
    ltq.dequantize_tokens(q, qp, getattr(cuda, dtype), out=out[:, first:first + K])
    want = cuda.from_numpy(values_f32(codes, scales, zeros)).to(getattr(cuda, dtype))
    got = out.cpu()
    assert cuda.equal(got[:, first:first + K], want)
    got[:, first:first + K] = 7.0
    assert (got == 7.0).all(), "columns outside the view were written"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (2, 15), (3, 16), (2, 17), (5, 512), (3, 513), (2, 8192), (700, 48)])
def test_dequantize_tokens(cuda, dtype, M, K):
    import ltq
    torch = cuda
    g = torch.Generator().manual_seed(K)
    codes = torch.randint(0, 256, (M, K), generator=g, dtype=torch.uint8)
    scale = torch.exp(torch.randn(M, generator=g))
    qp = torch.zeros(M, 8, dtype=torch.uint8)
    qp.view(torch.float32)[:, 0] = scale
    qp[:, 4] = torch.randint(0, 256, (M,), generator=g, dtype=torch.uint8)
    if M > 1:
        qp.view(torch.float32)[1, 0] = float("nan")
    got = ltq.dequantize_tokens(codes.cuda(), qp.cuda(), getattr(torch, dtype)).cpu()
    want = (qp.view(torch.float32)[:, :1] * (codes.float() - qp[:, 4:5].float())).to(getattr(torch, dtype))
    assert torch.equal(got[0], want[0]) and (M < 3 or torch.equal(got[2:], want[2:]))
    if M > 1:
        assert torch.isnan(got[1]).all()


# ---- the product ----------------------------------------------------------------------------------------------------------

def product_case(torch, seed, M, N, K, bias):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randint(0, 256, s, generator=g, dtype=torch.uint8)  # noqa: E731

    def pairs(n):
        p = torch.zeros(n, 8, dtype=torch.uint8)
        p.view(torch.float32)[:, 0] = 0.01 * torch.exp(0.5 * torch.randn(n, generator=g))
        p[:, 4] = r(n)
        return p
    c = dict(a=r(M, K), w=r(N, K), qa=pairs(M), qw=pairs(N), bias=torch.randn(N, generator=g) if bias else None)
    if M > 2:
        c["qa"][1, 4], c["qa"][2, 4] = 0, 255     # zero points at the ends of the range
    if N > 2:
        c["qw"][0, 4], c["qw"][2, 4] = 255, 0
    return c


def product_want(torch, c, dtype, relu):
    acc = (c["a"].double() - c["qa"][:, 4:5].double()) @ (c["w"].double() - c["qw"][:, 4:5].double()).t()   # exact: below 2^53
    y = acc.float() * c["qa"].view(torch.float32)[:, :1]
    y = y * c["qw"].view(torch.float32)[:, 0]
    if c["bias"] is not None:
        y = y + c["bias"]
    if relu:
        y = torch.where(y < 0, torch.zeros(()), y)
    return y.to(getattr(torch, dtype))


def run_product(ltq, c, dtype, flags, out=None):
    h = ltq.LayerHandle(0, c["a"].shape[1], c["w"].shape[0])
    h.set_weights(c["w"].cuda())
    h.set_channel_qparams(c["qw"].cuda(), None if c["bias"] is None else c["bias"].cuda())
    sums = c["a"].int().sum(1, dtype=c["a"].int().dtype).cuda()
    y = h.forward_tokens(c["a"].cuda(), c["qa"].cuda(), sums, dtype, flags, out=out)
    h.check()
    return y


SHAPES = [(1, 1, 1), (1, 8, 128), (3, 130, 256), (16, 264, 1024), (17, 64, 48), (5, 7, 3), (33, 31, 100), (128, 128, 128), (129, 257, 272),
          (64, 4099, 256), (300, 640, 512), (1, 11008, 512), (16, 2048, 4096),
          # few tiles: K divided over clusters, one, two and four lines of K per copy, rows that are no multiple of eight
          (77, 1024, 4096), (32, 200, 8192), (20, 1030, 2048), (100, 264, 8192), (40, 100, 2064), (33, 520, 5008), (130, 96, 4096), (24, 4096, 1152)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_is_exact_up_to_its_float_steps(cuda, dtype, M, N, K):
    import ltq
    for bias, relu in ((False, False), (True, True)):
        c = product_case(cuda, M * 7 + N + K, M, N, K, bias)
        got = run_product(ltq, c, getattr(cuda, dtype), ltq.FLAG_RELU if relu else 0)
        assert cuda.equal(got.cpu(), product_want(cuda, c, dtype, relu))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("flag,kernel,M,N,K", [("FLAG_FORCE_SIMT", "gemm_simt", 70, 90, 64), ("FLAG_FORCE_TC_SINGLE", "gemm_small_kernel", 200, 500, 144),
                                               ("FLAG_FORCE_TC_PAIR", "gemm_tc_pair_kernel", 333, 777, 208), ("FLAG_FORCE_SKINNY", "gemv_kernel", 11, 1000, 384),
                                               ("FLAG_FORCE_TC_PAIR", "gemm_tc_pair_kernel", 2048, 2048, 256), ("FLAG_FORCE_TC_PAIR", "gemm_tc_pair_kernel", 700, 2051, 384)])
def test_every_kernel_gives_the_same_product(cuda, dtype, flag, kernel, M, N, K):
    import ltq
    c = product_case(cuda, N, M, N, K, True)
    flags = getattr(ltq, flag) | (ltq.FLAG_FORCE_TC if "TC" in flag else 0)
    got = run_product(ltq, c, getattr(cuda, dtype), flags)
    assert ltq.last_kernel().startswith(kernel)
    assert cuda.equal(got.cpu(), product_want(cuda, c, dtype, False))


def test_product_writes_strided_rows_only(cuda):
    import ltq
    for M, N, K, ld in ((5, 24, 128, 40), (200, 130, 64, 131), (300, 256, 64, 264)):
        c = product_case(cuda, M, M, N, K, True)
        buf = cuda.full((M, ld), 3.0, dtype=cuda.bfloat16, device="cuda")
        run_product(ltq, c, cuda.bfloat16, 0, out=buf[:, :N])
        got = buf.cpu()
        assert cuda.equal(got[:, :N], product_want(cuda, c, "bfloat16", False)) and (got[:, N:] == 3.0).all()


def test_largest_inner_size_cannot_overflow(cuda):
    """in_features 33025 with every factor at the end of its range: 33025 * 255 * 255 < 2^31."""
    import ltq
    K = 33025
    c = product_case(cuda, 1, 18, 9, K, False)
    c["a"][:] = 255
    c["w"][:] = 255
    c["qa"][:, 4] = 0
    c["qw"][:, 4] = 0
    c["a"][1] = 0
    c["qa"][1, 4] = 255
    assert cuda.equal(run_product(ltq, c, cuda.float32, 0).cpu(), product_want(cuda, c, "float32", False))
    h = ltq.LayerHandle(0, K + 1, 1)
    h.set_weights(cuda.zeros(1, K + 1, dtype=cuda.uint8, device="cuda"))
    with pytest.raises(ltq.LtqError) as e:
        h.set_channel_qparams(cuda.zeros(1, 8, dtype=cuda.uint8, device="cuda"))
    assert e.value.status == -2


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 40, 4096), (4, 264, 1000), (16, 1030, 1024), (77, 130, 1021), (200, 300, 77), (300, 4096, 512)])
def test_forward_float_is_quantise_then_product(cuda, oracle, dtype, M, N, K):
    """Any width (those that are not multiples of 16 go through padded codes and weights), strided input rows."""
    import ltq
    torch = cuda
    c = product_case(torch, K, M, N, K, True)
    x = rows_of(torch, M, M, K + 24, dtype)
    layer = ltq.FullyConnected_t(c["w"].cuda(), c["qw"].cuda(), c["bias"].cuda())
    dev = x.cuda()[:, 8:8 + K]
    got = layer.forward(dev)
    codes, scales, zeros = oracle_rows(oracle, x[:, 8:8 + K])
    c["a"] = torch.from_numpy(codes)
    c["qa"] = torch.zeros(M, 8, dtype=torch.uint8)
    c["qa"].view(torch.float32)[:, 0] = torch.from_numpy(scales)
    c["qa"][:, 4] = torch.from_numpy(zeros)
    assert got.dtype == x.dtype and torch.equal(got.cpu(), product_want(torch, c, dtype, False))
    folded = layer.forward(dev.reshape(1, M, K))
    assert folded.shape == (1, M, N) and torch.equal(folded[0], got)
    layer.set_output(relu=True)
    assert torch.equal(layer.forward(dev).cpu(), product_want(torch, c, dtype, True))
    mixed = layer._handle.forward_float(dev, torch.float32)
    assert torch.equal(mixed.cpu(), product_want(torch, c, "float32", False))


def test_a_token_that_is_not_finite_shows_in_its_row_only(cuda):
    import ltq
    x = cuda.randn(20, 256).bfloat16()
    clean = x.clone()
    x[3, 17] = float("nan")
    x[18, 0] = float("-inf")
    layer = ltq.FullyConnected_t.from_float(cuda.randn(48, 256).cuda())
    for relu in (False, True):
        layer.set_output(relu=relu)
        y, want = layer.forward(x.cuda()), layer.forward(clean.cuda())
        assert cuda.isnan(y[[3, 18]]).all()
        keep = [i for i in range(20) if i not in (3, 18)]
        assert cuda.equal(y[keep], want[keep])


def test_from_float_and_weights_rebound(cuda, oracle):
    import ltq
    w = cuda.randn(33, 500)
    codes, scales, zeros = oracle_rows(oracle, w)
    layer = ltq.FullyConnected_t.from_float(w.cuda(), cuda.zeros(33).cuda())
    assert np.array_equal(layer.get_weights().cpu().numpy(), codes)
    assert layer.is_using_bias()
    h = layer._handle
    h.set_weights(layer.get_weights())
    with pytest.raises(ltq.LtqError, match="ltq_layer_set_channel_qparams"):
        layer.forward(cuda.randn(2, 500).cuda())
    h.set_channel_qparams(layer.weight_qparams_, None)
    assert layer.forward(cuda.randn(2, 500).cuda()).shape == (2, 33)


def test_other_stream_and_captured_replay(cuda):
    """The call runs on the caller's stream; a captured one follows its inputs and matches the eager one bit for bit."""
    import ltq
    torch = cuda
    layer = ltq.FullyConnected_t.from_float(torch.randn(96, 384).cuda(), torch.randn(96).cuda())
    x = torch.randn(9, 384).half().cuda()
    want = layer.forward(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer.forward(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    static = x.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer.forward(static)
    for seed in range(3):
        new = torch.randn(9, 384, generator=torch.Generator().manual_seed(seed)).half().cuda()
        static.copy_(new)
        graph.replay()
        assert torch.equal(y, layer.forward(new))


def test_no_tokens(cuda):
    import ltq
    layer = ltq.FullyConnected_t.from_float(cuda.randn(16, 64).cuda())
    assert layer.forward(cuda.empty(0, 64, device="cuda")).shape == (0, 16)
    q, qp, sums = ltq.quantize_tokens(cuda.empty(0, 64, device="cuda"))
    assert q.shape == (0, 64) and qp.shape == (0, 8) and sums.shape == (0,)
    assert ltq.dequantize_tokens(q, qp).shape == (0, 64)


def test_refusals(cuda):
    import ltq
    torch = cuda
    x = torch.randn(4, 64).cuda()
    q, qp, sums = ltq.quantize_tokens(x)
    layer = ltq.FullyConnected_t.from_float(torch.randn(16, 64).cuda())
    for bad in (lambda: ltq.quantize_tokens(x.double()), lambda: ltq.quantize_tokens(x.cpu()), lambda: ltq.quantize_tokens(x.t()),
                lambda: ltq.quantize_tokens(x[0]), lambda: ltq.quantize_tokens(x[:1].expand(4, 64)), lambda: ltq.quantize_tokens(x, q=q[:2]),
                lambda: ltq.dequantize_tokens(q, qp[:2]), lambda: ltq.dequantize_tokens(q, qp, torch.float64),
                lambda: ltq.dequantize_tokens(q.t(), qp), lambda: layer.forward(x[:, :32]), lambda: layer.forward(x.cpu()),
                lambda: layer.forward(x.double()), lambda: layer._handle.forward_tokens(q, qp[:1], sums),
                lambda: layer._handle.forward_tokens(q, qp, sums[:1]), lambda: layer._handle.forward_tokens(q, qp, sums, torch.float64),
                lambda: layer._handle.forward_tokens(q, qp, sums, out=torch.empty(4, 15, device="cuda")),
                lambda: layer._handle.set_channel_qparams(qp), lambda: ltq.FullyConnected_t(x, qp)):
        with pytest.raises(ValueError):
            bad()
