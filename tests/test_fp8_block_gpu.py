"""Block-scaled FP8 kernels against the 64-bit oracle: codes and scales bit for
bit, products within the oracle's bounds."""
import math

import pytest
import torch

from oracle import fp8_block as O

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(seed, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * std).to(dtype)


def weights(seed, E, N, K):
    """Codes and scales of random weights, made by the oracle."""
    q, s = O.quantize_blocks(randn(seed, E, N, K, std=0.02).double())
    return q.float().to(F8), s.float()


def same(t, ref):
    """Equal values, NaN where the reference has NaN."""
    a, b = t.double(), ref.double()
    return bool(torch.all((a == b) | (a.isnan() & b.isnan())))


# ------------------------------------------------------------------ quantizers
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (1, 2816), (3, 127), (5, 129), (17, 704), (300, 2816), (2, 8200),
                                 (1, 20000), (2000, 136), (9, 1000)])
def test_quantize_rows(M, K, dtype):
    from aeo_quant_b200.gpu.quant import quantize_fp8_activation_blocks
    x = randn(M + K, M, K, std=3.0, dtype=dtype)
    q, s = quantize_fp8_activation_blocks(x)
    assert q.dtype == F8 and q.shape == (M, K) and s.dtype == torch.float32 and s.shape == (M, -(-K // 128))
    rq, rs = O.quantize_rows(x.double())
    assert same(q, rq) and same(s, rs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E,N,K", [(1, 1, 1), (2, 128, 128), (1, 130, 260), (3, 1408, 704), (1, 7, 1000), (2, 300, 129)])
def test_quantize_weights(E, N, K, dtype):
    from aeo_quant_b200.gpu.quant import quantize_2d_to_fp8_block, quantize_3d_to_fp8_block
    w = randn(N + K, E, N, K, std=0.02, dtype=dtype)
    q, s = quantize_3d_to_fp8_block(w)
    assert q.dtype == F8 and q.shape == w.shape and s.shape == (E, -(-N // 128), -(-K // 128))
    rq, rs = O.quantize_blocks(w.double())
    assert same(q, rq) and same(s, rs)
    q0, s0 = quantize_2d_to_fp8_block(w[0])
    assert same(q0, rq[0]) and same(s0, rs[0])


def test_quantize_extremes():
    from aeo_quant_b200.gpu.quant import quantize_2d_to_fp8_block, quantize_fp8_activation_blocks
    inf, nan = float("inf"), float("nan")
    x = randn(1, 12, 300, dtype=torch.float32)
    x[0] = 0
    x[1, :128] = 1e-38
    x[2] *= 1e-31
    x[3] *= 1e36
    x[4, 5], x[4, 200] = inf, -inf
    x[5, 130] = nan
    x[6, :] = torch.finfo(torch.float32).min
    x[7, :128] = -0.0
    x[8, 0], x[8, 1] = 448.0, 464.0 / 512
    x[9] = torch.arange(300, device="cuda") / 16.0           # many ties
    x[10] = 7.0 * torch.arange(300, device="cuda") / 32.0
    x[11] = torch.finfo(torch.float32).tiny
    q, s = quantize_fp8_activation_blocks(x)
    rq, rs = O.quantize_rows(x.double())
    assert same(s, rs)
    ok = ~rs.repeat_interleave(128, 1)[:, :300].isnan()
    assert same(q.double()[ok], rq[ok]) and bool(q.float()[~ok].isnan().all())
    q, s = quantize_2d_to_fp8_block(x)
    assert bool(s.isnan().any()) and not bool(s.isnan().all())


def test_quantize_strides_and_empty():
    from aeo_quant_b200.gpu.quant import quantize_3d_to_fp8_block, quantize_fp8_activation_blocks
    big = randn(2, 40, 1000)
    for x in (big[:, :256], big[:, 3:259], big[::3, 8:520], big.t()[:130], big[0], big[:, None, 16:160],
              big[:1, :200].expand(6, 200), big.view(4, 10, 1000)[:, :, :136]):
        q, s = quantize_fp8_activation_blocks(x)
        rq, rs = O.quantize_rows(x.reshape(-1, x.shape[-1]).double())
        assert q.shape == x.shape and same(q.reshape(rq.shape), rq) and same(s.reshape(rs.shape), rs)
    w = big.view(4, 10, 1000)[:, :, 7:207].transpose(1, 2)
    q, s = quantize_3d_to_fp8_block(w)
    rq, rs = O.quantize_blocks(w.double())
    assert same(q, rq) and same(s, rs)
    q, s = quantize_fp8_activation_blocks(big[:0])
    assert q.shape == (0, 1000) and s.shape == (0, 8)
    q, s = quantize_fp8_activation_blocks(big[:, :0])
    assert q.shape == (40, 0) and s.shape == (40, 0)
    assert quantize_3d_to_fp8_block(big.view(4, 10, 1000)[:0])[0].shape == (0, 10, 1000)


# ---------------------------------------------------------------------- linear
def check_linear(x, w, ws, bias=None, out_dtype=torch.bfloat16):
    from aeo_quant_b200.gpu.fp8_block_matmul import fp8_block_linear
    y = fp8_block_linear(x, w, ws, bias, out_dtype=out_dtype)
    K = x.shape[-1]
    ref, tol = O.linear(x.reshape(-1, K).double(), w.double(), ws.double(), None if bias is None else bias.double(),
                        out_dtype == torch.bfloat16)
    assert y.dtype == out_dtype and y.shape == (*x.shape[:-1], w.shape[0])
    err = (y.reshape(ref.shape).double() - ref).abs()
    worst = float((err / tol.clamp_min(1e-30)).max()) if err.numel() else 0.0
    assert worst <= 1, f"{worst} of the bound"
    return y


@pytest.mark.parametrize("M", [1, 2, 3, 7, 8, 9, 16, 17, 31, 33, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("N,K", [(1408, 2816), (2112, 704), (100, 16), (1, 144), (257, 272)])
def test_linear_sizes(M, N, K):
    w, s = weights(N + K, 1, N, K)
    check_linear(randn(M, M, K), w[0], s[0])


@pytest.mark.parametrize("M,N,K", [(4096, 1408, 2816), (5000, 257, 144), (1500, 4000, 1040), (40, 30000, 256),
                                   (1, 40000, 512), (20000, 384, 128), (40, 8192, 2048), (8, 6000, 4096),
                                   (2100, 1408, 272), (1, 1000, 16400)])
def test_linear_large(M, N, K):
    w, s = weights(N + K, 1, N, K)
    check_linear(randn(M, M, K), w[0], s[0])


@pytest.mark.parametrize("M", [1, 5, 40, 200])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_linear_types_and_bias(M, dtype, out_dtype):
    for N, K in ((384, 272), (203, 704)):
        w, s = weights(7, 1, N, K)
        check_linear(randn(3, M, K, dtype=dtype), w[0], s[0], randn(4, N), out_dtype)


def test_linear_scales_vary_by_block():
    """Scales of very different size in neighbouring blocks: each has to meet its own block."""
    g = gen(5)
    for M in (1, 6, 50, 500):
        N, K = 700, 1200
        w, s = weights(8, 1, N, K)
        s = torch.exp2(torch.randint(-20, 20, s.shape, generator=g, device="cuda").float())
        x = randn(M, M, K, dtype=torch.float32) * torch.exp2(
            torch.randint(-20, 20, (M, 10), generator=g, device="cuda").float()).repeat_interleave(128, 1)[:, :K]
        check_linear(x, w[0], s[0], out_dtype=torch.float32)


def test_linear_special_rows():
    """A NaN or infinite row stays its own; zero rows give zero (or the bias)."""
    from aeo_quant_b200.gpu.fp8_block_matmul import fp8_block_linear
    w, s = weights(9, 1, 300, 400)
    for M in (6, 40, 200):
        x = randn(10, M, 400)
        x[1, 390], x[2, 3], x[3] = float("nan"), float("inf"), 0
        y = fp8_block_linear(x, w[0], s[0])
        keep = torch.ones(M, dtype=torch.bool, device="cuda")
        keep[1:3] = False
        assert bool(y[1:3].isnan().all()) and bool((y[3] == 0).all())
        assert torch.equal(y[keep], check_linear(x[keep], w[0], s[0])) or M < 20
        b = randn(11, 300)
        assert torch.equal(fp8_block_linear(x, w[0], s[0], b)[3], b)


def test_linear_strides_shapes_prequantized():
    from aeo_quant_b200.gpu.fp8_block_matmul import fp8_block_linear, fp8_block_linear_prequantized
    from aeo_quant_b200.gpu.quant import quantize_fp8_activation_blocks
    w, s = weights(12, 1, 500, 256)
    big = randn(13, 60, 900)
    for x in (big[:, :256], big[:, 5:261], big[::2, 8:264], big[:, 128:384].reshape(3, 20, 256), big[0, :256],
              big[:1, :256].expand(4, 256), big.t()[:256, :].t()):
        check_linear(x, w[0], s[0])
    check_linear(big[:9, :256], w[0].t().contiguous().t(), s[0].t().contiguous().t())
    check_linear(big[:9, :256], w[0][100:], s[0][:4])            # 16-byte aligned start inside a storage
    assert fp8_block_linear(big[:0, :256], w[0], s[0]).shape == (0, 500)
    for M in (1, 30, 60):
        xq, xs = quantize_fp8_activation_blocks(big[:M, :256])
        y = fp8_block_linear_prequantized(xq, xs, w[0], s[0], out_dtype=torch.float32)
        ref, tol = O.linear(big[:M, :256].double(), w[0].double(), s[0].double(), out_bf16=False)
        assert bool(((y.double() - ref).abs() <= tol).all())


def test_linear_same_bits_again_and_in_a_graph():
    from aeo_quant_b200.gpu.fp8_block_matmul import fp8_block_linear
    w, s = weights(14, 1, 1408, 2816)
    for M in (1, 4, 48, 700):
        x = randn(M, M, 2816)
        want = fp8_block_linear(x, w[0], s[0])
        assert all(torch.equal(want, fp8_block_linear(x, w[0], s[0])) for _ in range(3))
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got = fp8_block_linear(x, w[0], s[0])
        st.synchronize()
        assert torch.equal(want, got)
        buf = torch.zeros_like(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fp8_block_linear(buf, w[0], s[0])
        for k in range(2):
            buf.copy_(x * (k + 1))
            graph.replay()
            assert torch.equal(out, fp8_block_linear(x * (k + 1), w[0], s[0]))


# --------------------------------------------------------------------- experts
def routing(seed, T, E, k, dropped=0.0):
    g = gen(seed)
    ids = torch.rand(T, E, generator=g, device="cuda").topk(k, -1).indices
    w = torch.softmax(torch.randn(T, k, generator=g, device="cuda"), -1)
    if dropped:
        ids = ids.masked_fill(torch.rand(T, k, generator=g, device="cuda") < dropped, E)
    return ids, w


def check_experts(x, ids, w, gu, gs, dw, ds, act):
    from aeo_quant_b200.bridges.gemma4.moe_ops import fp8_block_experts
    y = fp8_block_experts(x, ids, w, gu, gs, dw, ds, activation=act)
    ref, tol = O.experts(x.double(), ids, w.double(), gu.double(), gs.double(), dw.double(), ds.double(), act)
    assert y.shape == x.shape and y.dtype == torch.bfloat16
    err = (y.double() - ref).abs()
    worst = float((err / tol.clamp_min(1e-30)).max()) if err.numel() else 0.0
    assert worst <= 1, f"{worst} of the bound"
    # That bound lets every error add up. As a whole the error is that of two
    # bf16 roundings (the experts' outputs, the sum), each of at most 2^-8 /
    # sqrt(3) of the value in the mean square: 3.2e-3 together, and a few
    # codes of h that fall the other way.
    assert float(err.norm()) <= 5e-3 * float(ref.norm())
    return y


@pytest.mark.parametrize("T", [1, 2, 5, 16, 40, 200])
@pytest.mark.parametrize("E,k,H,I,act", [(16, 8, 2816, 704, "gelu_pytorch_tanh"), (4, 1, 256, 64, "silu"),
                                         (8, 2, 400, 192, "silu"), (40, 6, 528, 320, "gelu_pytorch_tanh"),
                                         (1, 1, 128, 128, "silu")])
def test_experts_sizes(T, E, k, H, I, act):
    gu, gs = weights(E + H, E, 2 * I, H)
    dw, ds = weights(E + I, E, H, I)
    check_experts(randn(T, T, H), *routing(T, T, E, k), gu, gs, dw, ds, act)


@pytest.mark.parametrize("T,E,k,H,I", [(1500, 8, 2, 512, 256), (300, 128, 8, 256, 128), (700, 3, 3, 1040, 448),
                                       (900, 16, 8, 272, 192), (600, 128, 8, 144, 64), (70, 1024, 4, 64, 64),
                                       (2000, 1024, 3, 64, 64), (5000, 4, 1, 128, 64), (30, 4, 4, 16, 64),
                                       (4097, 32, 1, 16, 128)])
def test_experts_many_tokens(T, E, k, H, I):
    gu, gs = weights(E + H, E, 2 * I, H)
    dw, ds = weights(E + I, E, H, I)
    check_experts(randn(T, T, H), *routing(T, T, E, k, 0.1), gu, gs, dw, ds, "silu")


def test_experts_ids_weights_and_edges():
    from aeo_quant_b200.bridges.gemma4.moe_ops import fp8_block_experts
    E, H, I, k = 8, 256, 128, 4
    gu, gs = weights(20, E, 2 * I, H)
    dw, ds = weights(21, E, H, I)
    for T in (1, 3, 50, 150):
        x = randn(T, T, H)
        ids, w = routing(T, T, E, k)
        want = check_experts(x, ids, w, gu, gs, dw, ds, "silu")
        assert torch.equal(want, fp8_block_experts(x, ids.int(), w, gu, gs, dw, ds, "silu"))
        wb = w.bfloat16()
        assert torch.equal(fp8_block_experts(x, ids, wb, gu, gs, dw, ds, "silu"),
                           fp8_block_experts(x, ids, wb.float(), gu, gs, dw, ds, "silu"))
        assert bool((fp8_block_experts(x, torch.full_like(ids, E), w, gu, gs, dw, ds) == 0).all())
        assert bool((fp8_block_experts(x, torch.full_like(ids, -1), w, gu, gs, dw, ds) == 0).all())
        one = torch.full_like(ids, 3)                        # every slot the same expert
        check_experts(x, one, w, gu, gs, dw, ds, "silu")
        odd = ids.clone()
        odd[:, 1], odd[0, 0] = -7, 1 << 20                   # skipped ids in between
        check_experts(x, odd, w, gu, gs, dw, ds, "silu")
        if T > 2:
            bad = x.clone()
            bad[1, 7] = float("nan")                         # one token's NaN stays its own
            got = fp8_block_experts(bad, ids, w, gu, gs, dw, ds, "silu")
            assert bool(got[1].isnan().all())
            assert torch.equal(got[[0, 2]], want[[0, 2]])
    assert fp8_block_experts(x[:0], ids[:0], w[:0], gu, gs, dw, ds).shape == (0, H)


def test_experts_strides_stream_graph():
    from aeo_quant_b200.bridges.gemma4.moe_ops import fp8_block_experts
    E, H, I, k = 16, 512, 192, 4
    gu, gs = weights(22, E, 2 * I, H)
    dw, ds = weights(23, E, H, I)
    for T in (1, 6, 130):
        big = randn(T, T, 2 * H + 8)
        ids, w = routing(T, T, E, 2 * k)
        for x in (big[:, :H], big[:, 3:3 + H], big[:, 8:8 + H]):
            check_experts(x, ids[:, ::2], w[:, ::2], gu, gs, dw, ds, "silu")
        x, i, v = big[:, :H].contiguous(), ids[:, :k].contiguous(), w[:, :k].contiguous()
        want = fp8_block_experts(x, i, v, gu, gs, dw, ds)
        assert all(torch.equal(want, fp8_block_experts(x, i, v, gu, gs, dw, ds)) for _ in range(3))
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        outs = []
        for st in (s1, s2):                                  # two calls at once
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                outs += [fp8_block_experts(x, i, v, gu, gs, dw, ds) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(want, o) for o in outs)
        bx, bi = torch.zeros_like(x), torch.zeros_like(i)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fp8_block_experts(bx, bi, v, gu, gs, dw, ds)
        bx.copy_(x)
        bi.copy_(i)
        graph.replay()
        assert torch.equal(out, want)


# ------------------------------------------------------- C entry, sizes, streams
@pytest.mark.parametrize("out_dt", [0, 2])
@pytest.mark.parametrize("M,N,K", [(1, 130, 256), (5, 200, 144), (40, 130, 256), (300, 400, 256), (257, 127, 400)])
@pytest.mark.parametrize("pad,shift", [(8, 0), (3, 0), (8, 1)])
def test_linear_into_a_larger_output(M, N, K, out_dt, pad, shift):
    """Rows of a larger output, aligned for wide stores or not: what lies
    between and behind the product's values stays as it was."""
    from aeo_quant_b200 import _capi as A
    from aeo_quant_b200.gpu.fp8_block_matmul import fp8_block_linear
    dt = torch.bfloat16 if out_dt == 0 else torch.float32
    x = randn(21, M, K)
    w, s = weights(22, 1, N, K)
    ldc = (N + 7) // 8 * 8 + pad
    buf = torch.full(((M + 2) * ldc + shift,), 7.0, dtype=dt, device="cuda")
    out = buf[shift:].view(M + 2, ldc)
    n = A.load().aeoq_fp8_block_linear_workspace_size(M, N, K)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    A.check(A.load().aeoq_fp8_block_linear(x.data_ptr(), A.dtype_code(x.dtype), K, M, w[0].data_ptr(),
                                           s[0].data_ptr(), N, K, None, out.data_ptr(), out_dt, ldc, ws.data_ptr(), n,
                                           A.err_ptr(0), A.raw_stream(torch.cuda.current_device())))
    assert torch.equal(out[:M, :N], fp8_block_linear(x, w[0], s[0], out_dtype=dt))
    assert bool((out[:M, N:] == 7).all()) and bool((out[M:] == 7).all()) and bool((buf[:shift] == 7).all())


def test_rows_past_32_bit_offsets():
    """Input rows that start past 2^31 elements."""
    from aeo_quant_b200.gpu.fp8_block_matmul import fp8_block_linear
    from aeo_quant_b200.gpu.quant import quantize_fp8_activation_blocks
    w, s = weights(23, 1, 200, 512)
    for M, ld in ((4, 1 << 30), (20, 1 << 27), (300, 1 << 23)):
        x = torch.empty((M - 1) * ld + 512, dtype=torch.bfloat16, device="cuda").as_strided((M, 512), (ld, 1))
        x.copy_(randn(24, M, 512))
        near = x.contiguous()
        for a, b in zip(quantize_fp8_activation_blocks(x), quantize_fp8_activation_blocks(near)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert torch.equal(fp8_block_linear(x, w[0], s[0]), fp8_block_linear(near, w[0], s[0]))
        del x


def test_experts_past_32_bit_offsets():
    """Experts whose weights start past 2^31 bytes, and tokens whose experts'
    outputs start past 2^31 values: the same bits as from a small layer."""
    from aeo_quant_b200.bridges.gemma4.moe_ops import fp8_block_experts
    E, H, I = 9, 16384, 8192
    g = gen(25)

    def codes(*shape):
        return torch.randint(0, 0x60, shape, dtype=torch.uint8, device="cuda", generator=g).view(F8)

    def scales(E, n, k):
        return torch.rand(E, -(-n // 128), -(-k // 128), device="cuda", generator=g) * 1e-4
    gu, gs, dw, ds = codes(E, 2 * I, H), scales(E, 2 * I, H), codes(E, H, I), scales(E, H, I)
    for T in (1, 36, 250):          # each of the three forms: 2 T pairs on 9 or 2 experts
        x = randn(26, T, H)
        ids = torch.tensor([[E - 1, E - 2]], device="cuda").repeat(T, 1)
        w = torch.rand(T, 2, device="cuda", generator=g)
        big = fp8_block_experts(x, ids, w, gu, gs, dw, ds, activation="silu")
        small = fp8_block_experts(x, ids - (E - 2), w, *(t[E - 2:] for t in (gu, gs, dw, ds)), activation="silu")
        assert torch.equal(big, small) and bool(torch.isfinite(big).all())
    del gu, dw
    I, T, n = 64, 70000, 100
    gu, gs, dw, ds = codes(2, 2 * I, H), scales(2, 2 * I, H), codes(2, H, I), scales(2, H, I)
    x = randn(27, T, H)
    ids = torch.tensor([[0, 1]], device="cuda").repeat(T, 1)
    w = torch.rand(T, 2, device="cuda", generator=g)
    big = fp8_block_experts(x, ids, w, gu, gs, dw, ds)
    assert torch.equal(big[-n:], fp8_block_experts(x[-n:], ids[-n:], w[-n:], gu, gs, dw, ds))


def test_experts_on_two_streams_at_once():
    """Calls that overlap, eager and as two captured graphs, share nothing."""
    from aeo_quant_b200.bridges.gemma4.moe_ops import fp8_block_experts
    E, k, H, I = 16, 4, 512, 128
    gu, gs = weights(28, E, 2 * I, H)
    dw, ds = weights(29, E, H, I)
    jobs = []
    for i, T in enumerate((3, 40, 700, 2, 55, 900)):
        ids, w = routing(30 + i, T, E, k)
        x = randn(40 + i, T, H)
        jobs.append((x, ids, w, fp8_block_experts(x, ids, w, gu, gs, dw, ds)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[] for _ in jobs]
    for _ in range(5):
        for j, (x, ids, w, _) in enumerate(jobs):
            with torch.cuda.stream(streams[j]):
                got[j].append(fp8_block_experts(x, ids, w, gu, gs, dw, ds))
    torch.cuda.synchronize()
    for j, (_, _, _, want) in enumerate(jobs):
        assert all(torch.equal(want, y) for y in got[j])
    graphs = []
    for x, ids, w, _ in jobs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fp8_block_experts(x, ids, w, gu, gs, dw, ds)
        graphs.append((graph, y))
    for _, y in graphs:
        y.zero_()
    torch.cuda.synchronize()
    for st, (graph, _) in zip(streams, graphs):
        with torch.cuda.stream(st):
            graph.replay()
    torch.cuda.synchronize()
    for (_, y), (_, _, _, want) in zip(graphs, jobs):
        assert torch.equal(y, want)


# ------------------------------------------------------- one rounding per output
@pytest.mark.parametrize("T,E,k,H,I", [(4, 16, 8, 512, 256), (8, 40, 6, 528, 320), (40, 40, 6, 528, 320),
                                       (64, 128, 8, 1040, 192), (300, 8, 2, 512, 256), (700, 3, 3, 1040, 448)])
def test_experts_round_once(T, E, k, H, I):
    """A token's experts are summed in f32 and rounded once, whatever the
    number of tokens beside it: the layer's error is that of this rounding.

    Beyond it: f32 sums know h to about 2^-20 of a block's largest value, so
    one in 2^16 or so of its codes falls the other way, each by at most 2^-3
    of its value: 2^-11 in the mean square, against some 2^-9.2 of a bf16
    rounding: 1.04 of it together. A second rounding, of each expert's
    output, would make it 1.41."""
    from aeo_quant_b200.bridges.gemma4.moe_ops import fp8_block_experts
    gu, gs = weights(E + H, E, 2 * I, H)
    dw, ds = weights(E + I, E, H, I)
    x, (ids, w) = randn(T, T, H), routing(T, T, E, k)
    y = fp8_block_experts(x, ids, w, gu, gs, dw, ds, activation="silu")
    ref, _ = O.experts(x.double(), ids, w.double(), gu.double(), gs.double(), dw.double(), ds.double(), "silu")
    once = (ref.bfloat16().double() - ref).norm()
    assert float((y.double() - ref).norm()) <= 1.2 * float(once)


# ------------------------------------------------------ strongly negative gates
@pytest.mark.parametrize("T,E", [(1, 2), (100, 4), (300, 2)])
@pytest.mark.parametrize("act,gain", [("gelu_pytorch_tanh", 1.25), ("silu", 6.0), ("silu", 2.0 ** 60),
                                      ("gelu_pytorch_tanh", 2.0 ** 60)])
@pytest.mark.parametrize("I", [64, 192])
def test_experts_strongly_negative_gates(T, E, act, gain, I):
    """Where all of a block's gates are strongly negative, their tiny values
    set the block's scale and are kept with full codes. The operands are
    chosen so that gates and ups are exact: one value per row of x whose code
    and scale are exact (7 = 448 / 2^6), one product per sum."""
    from aeo_quant_b200.bridges.gemma4.moe_ops import fp8_block_experts
    H = 128
    x = torch.zeros(T, H, device="cuda", dtype=torch.bfloat16)
    x[:, 0] = 7.0
    gu = torch.zeros(E, 2 * I, H, device="cuda")
    gu[:, :I, 0] = -(1 + torch.randint(0, 7, (E, I), generator=gen(I), device="cuda") / 8)     # -1 ... -1.75
    gu[:, I:, 0] = (1 + torch.randint(0, 8, (E, I), generator=gen(I + 1), device="cuda") / 8)
    gs = torch.ones(E, -(-2 * I // 128), 1, device="cuda")
    gs[:, :I // 128] = gain
    if I % 128:
        gs[:, I // 128] = gain            # this block holds gates and ups
    dw = torch.zeros(E, H, I, device="cuda")
    dw[:, torch.arange(H), torch.arange(H) % I] = 1.0
    ds = torch.ones(E, 1, -(-I // 128), device="cuda")
    ids = torch.arange(T, device="cuda")[:, None] % E
    w = torch.ones(T, 1, device="cuda")
    y = fp8_block_experts(x, ids, w, gu.to(F8), gs, dw.to(F8), ds, activation=act).double()
    xd = O.value_rows(*O.quantize_rows(x.double()))
    full = torch.einsum("th,enh->ten", xd, O.value_blocks(gu.double(), gs.double()))
    g, u = full[torch.arange(T), ids[:, 0]].chunk(2, 1)
    # (as g * sigmoid: 1 + tanh cancels to 0 in 64 bits from about -7 on)
    h = g * torch.sigmoid(g if act == "silu" else 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)) * u
    hd = O.value_rows(*O.quantize_rows(h))[:, :128]
    ref = hd[:, torch.arange(H) % I]
    # a code may fall the other way (2^-3 of the value, or the smallest step,
    # 2^-9 of the scale), and the output is rounded to bf16
    step = h[:, :128].abs().amax(1, keepdim=True).clamp_min(1e-30) / 448 * 2.0 ** -9
    assert bool(((y - ref).abs() <= (2.0 ** -3 + 2.0 ** -7) * ref.abs() + 1.01 * step).all())


@pytest.mark.parametrize("T,E,k,H,I", [(1, 16, 9, 512, 1024), (1, 40, 32, 256, 832), (2, 40, 32, 272, 128),
                                       (3, 6, 2, 512, 2048), (1, 8, 2, 144, 3200), (5, 16, 12, 400, 960),
                                       (1, 1, 1, 64, 1600), (20, 8, 2, 528, 1792), (33, 8, 1, 256, 1344),
                                       (64, 4, 1, 512, 1088), (32, 2, 2, 1024, 896), (50, 1, 1, 256, 2112)])
@pytest.mark.parametrize("act", ["silu", "gelu_pytorch_tanh"])
def test_experts_few_pairs_wide_layers(T, E, k, H, I, act):
    """Up to 64 pairs: more slots than a CTA has warps, more of I than one
    round of loads, and layers of few experts that each take many pairs."""
    gu, gs = weights(E + H, E, 2 * I, H)
    dw, ds = weights(E + I, E, H, I)
    check_experts(randn(T, T, H), *routing(T, T, E, k), gu, gs, dw, ds, act)
    check_experts(randn(T, T, H), *routing(T + 1, T, E, k, 0.2), gu, gs, dw, ds, act)


@pytest.mark.parametrize("M", [4, 6, 8, 12, 30, 64, 200])
def test_linear_rows_beside_nan_and_infinite_ones(M):
    """The rows of a call that also holds NaN and infinite rows have the bits
    that they have beside finite ones."""
    from aeo_quant_b200.gpu.fp8_block_matmul import fp8_block_linear
    w, s = weights(31, 1, 300, 400)
    x = randn(32, M, 400)
    want = check_linear(x, w[0], s[0])
    bad = x.clone()
    bad[1, 390], bad[2, 3], bad[M - 1] = float("nan"), float("-inf"), float("inf")
    got = fp8_block_linear(bad, w[0], s[0])
    keep = torch.ones(M, dtype=torch.bool, device="cuda")
    keep[1:3] = keep[M - 1] = False
    assert bool(got[~keep].isnan().all()) and torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("N", [1, 8, 16, 24, 63, 72, 136, 264])
@pytest.mark.parametrize("M,K", [(64, 16), (130, 144), (400, 128)])
def test_linear_narrow_outputs(M, N, K):
    """Outputs narrower than a store's box of 64 columns, or a little wider."""
    w, s = weights(N + K, 1, N, K)
    check_linear(randn(M, M, K), w[0], s[0])
