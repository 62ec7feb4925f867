"""Block-scaled FP8 on the CPU: the oracle's rounding against torch's, and
every refusal that is decided before a GPU call."""
import math

import pytest
import torch

from oracle import fp8_block as O


@pytest.fixture(scope="module")
def lib():
    from aeo_quant_b200 import _capi
    return _capi.load()


def test_oracle_rounding_is_torchs():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    v = torch.sort(codes[codes.isfinite()]).values
    mid = (v[1:] + v[:-1]) / 2
    p = torch.cat([v, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20), torch.randn(10000, dtype=torch.float64) * 90])
    p = p.clamp(-448, 448).float()
    assert torch.equal(O.e4m3(p.double()).float(), p.to(torch.float8_e4m3fn).float())


def test_oracle_blocks_agree_with_whole_tensor_formula():
    x = torch.randn(5, 300, dtype=torch.float64)
    q, s = O.quantize_rows(x)
    assert q.shape == (5, 300) and s.shape == (5, 3)
    assert torch.all((O.value_rows(q, s) - x).abs() <= x.abs() * (2.0 ** -4 + 1e-6) + s.amax() * 2.0 ** -10)
    wq, ws = O.quantize_blocks(torch.randn(2, 130, 300, dtype=torch.float64))
    assert ws.shape == (2, 2, 3) and wq.abs().max() == 448


def test_quantizer_c_refusals(lib):
    f = lib.aeoq_fp8_block_quantize_rows
    assert f(None, 3, 4, 128, 128, None, 128, None, None) == -1 and b"dtype" in lib.aeoq_last_error()
    assert f(None, 0, 4, 128, 100, None, 128, None, None) == -1 and b"bad shape" in lib.aeoq_last_error()
    assert f(None, 0, 4, 128, 128, None, 128, None, None) == -1 and b"null" in lib.aeoq_last_error()
    assert f(None, 0, 0, 128, 128, None, 128, None, None) == 0
    g = lib.aeoq_fp8_block_quantize_weights
    assert g(None, 0, 70000, 128, 128, None, None, None) == -1 and b"65535" in lib.aeoq_last_error()
    assert g(None, 9, 1, 128, 128, 1, 1, None) == -1
    assert g(None, 0, 0, 128, 128, None, None, None) == 0


def test_linear_c_refusals(lib):
    def gemm(M=4, N=256, K=256, dt=0, ldc=256, p=None):
        return lib.aeoq_fp8_block_gemm(p, p, M, p, p, N, K, None, p, dt, ldc, None, None)
    assert gemm(K=24) == -1 and b"multiple of 16" in lib.aeoq_last_error()
    assert gemm(K=0) == -1
    assert gemm(M=-1) == -1
    assert gemm(dt=1) == -1 and b"output dtype" in lib.aeoq_last_error()
    assert gemm(ldc=255) == -1 and b"stride" in lib.aeoq_last_error()
    assert gemm() == -1 and b"null" in lib.aeoq_last_error()
    assert gemm(p=8) == -1 and b"aligned" in lib.aeoq_last_error()
    assert gemm(M=0) == 0 and gemm(N=0) == 0
    n = lib.aeoq_fp8_block_linear_workspace_size(33, 256, 272)
    assert n >= 33 * 272 + 33 * 3 * 4 and lib.aeoq_fp8_block_linear_workspace_size(0, 256, 256) == 0

    def linear(ws=None, bytes_=0, ldx=256, dt=0):
        return lib.aeoq_fp8_block_linear(16, dt, ldx, 40, 16, 16, 256, 256, None, 16, 0, 256, ws, bytes_, None, None)
    assert linear() == -3 and b"workspace" in lib.aeoq_last_error()
    assert linear(ws=256, bytes_=100) == -3
    assert linear(ws=257, bytes_=1 << 20) == -3
    assert linear(ldx=100) == -1 and linear(dt=4) == -1


def test_experts_c_refusals(lib):
    def fwd(T=4, k=8, E=16, H=256, I=128, idt=4, act=0, p=16, ws=None, n=0):
        return lib.aeoq_moe_fp8_block_forward(p, T, p, idt, p, k, p, p, p, p, E, H, I, act, p, ws, n, None, None)
    for bad, msg in ((dict(E=0), b"num_experts"), (dict(E=1025), b"num_experts"), (dict(k=0), b"top_k"),
                     (dict(k=33), b"top_k"), (dict(H=24), b"hidden"), (dict(I=96), b"intermediate"),
                     (dict(idt=0), b"int32/int64"), (dict(act=2), b"activation"), (dict(T=-1), b"token"),
                     (dict(p=None), b"null"), (dict(p=8), b"aligned")):
        assert fwd(**bad) == -1, bad
        assert msg in lib.aeoq_last_error(), bad
    assert fwd() == -3 and b"workspace" in lib.aeoq_last_error()
    assert fwd(T=0, p=None) == 0
    size = lib.aeoq_moe_fp8_block_workspace_size
    assert size(0, 8, 16, 256, 128) == 0
    assert size(64, 8, 128, 2816, 704) > size(4, 8, 128, 2816, 704) > 0


def test_python_refusals():
    from aeo_quant_b200 import AeoqError
    from aeo_quant_b200.bridges.gemma4 import moe_ops
    from aeo_quant_b200.gpu import fp8_block_matmul as F, quant as Q
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    w, s = torch.zeros(300, 256, dtype=torch.float8_e4m3fn), torch.zeros(3, 2)
    with pytest.raises(AeoqError):
        Q.quantize_fp8_activation_blocks(x)
    with pytest.raises(ValueError, match="unsupported dtype"):
        Q.quantize_fp8_activation_blocks(x.double())
    with pytest.raises(ValueError, match="expects a 3D"):
        Q.quantize_3d_to_fp8_block(x)
    with pytest.raises(ValueError, match="expects a 2D"):
        Q.quantize_2d_to_fp8_block(x[None])
    with pytest.raises(AeoqError):
        F.fp8_block_linear(x, w, s)
    for bad in (dict(w=w[None]), dict(w=w.float()), dict(s=torch.zeros(2, 2)), dict(s=s.double()), dict(x=x[:, :128]),
                dict(x=x.double()), dict(out_dtype=torch.float16), dict(bias=torch.zeros(300)),
                dict(bias=torch.zeros(10, dtype=torch.bfloat16))):
        a = dict(x=x, w=w, s=s, bias=None, out_dtype=torch.bfloat16)
        a.update(bad)
        with pytest.raises(ValueError):
            F.fp8_block_linear(a["x"], a["w"], a["s"], a["bias"], out_dtype=a["out_dtype"])
    with pytest.raises(ValueError, match="x_scale"):
        F.fp8_block_linear_prequantized(torch.zeros(4, 256, dtype=torch.float8_e4m3fn), torch.zeros(4, 3), w, s)
    with pytest.raises(ValueError, match="x_fp8"):
        F.fp8_block_linear_prequantized(x, torch.zeros(4, 2), w, s)
    E, H, I = 4, 256, 128
    a = dict(hidden=x, top_k_index=torch.zeros(4, 2, dtype=torch.int64), top_k_weights=torch.zeros(4, 2),
             gu=torch.zeros(E, 2 * I, H, dtype=torch.float8_e4m3fn), gu_scale=torch.zeros(E, 2, 2),
             dw=torch.zeros(E, H, I, dtype=torch.float8_e4m3fn), dw_scale=torch.zeros(E, 2, 1))
    with pytest.raises(AeoqError):
        moe_ops.fp8_block_experts(**a)
    for bad in (dict(hidden=x.float()), dict(hidden=x[0]), dict(gu=a["gu"][0]), dict(dw=a["dw"][:, :128]),
                dict(gu=a["gu"].float()), dict(gu_scale=torch.zeros(E, 2, 1)), dict(dw_scale=a["dw_scale"].half()),
                dict(top_k_index=torch.zeros(4, 3, dtype=torch.int64)), dict(top_k_index=torch.zeros(4, 2)),
                dict(top_k_weights=torch.zeros(4, 2, dtype=torch.int64)), dict(activation="relu"),
                dict(gu=a["gu"].transpose(1, 2).contiguous().transpose(1, 2)), dict(hidden=x[:, :128])):
        with pytest.raises(ValueError):
            moe_ops.fp8_block_experts(**{**a, **bad})


def test_dequantize_inverts():
    from aeo_quant_b200.gpu import quant as Q
    w = torch.randn(2, 150, 200, dtype=torch.float64)
    q, s = O.quantize_blocks(w)
    got = Q.dequantize_from_fp8_block(q.float().to(torch.float8_e4m3fn), s.float())
    assert torch.allclose(got.double(), O.value_blocks(q, s), rtol=1e-6) and math.isfinite(float(got.sum()))
    q, s = O.quantize_rows(w[0])
    got = Q.dequantize_fp8_activation_blocks(q.float().to(torch.float8_e4m3fn), s.float())
    assert torch.allclose(got.double(), O.value_rows(q, s), rtol=1e-6)


def test_form_of_few_pairs_goes_by_what_is_read_again(lib):
    """Up to 64 pairs an expert's weights are streamed once per pair, or the
    pairs are grouped by expert: by the bytes that streaming would read again.
    The forms differ in their workspace: h alone, against (among others) an
    f32 output row per pair."""
    def streams(T, k, E, H, I):
        n, h = lib.aeoq_moe_fp8_block_workspace_size(T, k, E, H, I), 4 * T * k * I
        assert n == -(-h // 256) * 256 or n >= 4 * T * k * H
        return n < 4 * T * k * H
    for E, k in ((1, 1), (8, 2), (16, 4), (64, 6), (128, 8), (1024, 32)):
        assert streams(1, k, E, 2816, 704)                 # one token: no expert twice
        assert not streams(64 // k + 1, k, E, 2816, 704)
    # a layer of 128 experts: its few pairs are almost all of other experts
    assert streams(4, 8, 128, 2816, 704) and streams(6, 8, 128, 2816, 704)
    # few experts: each of them would be read 8, 16, 32 and 64 times
    assert not any(streams(*c, 2816, 704) for c in ((32, 2, 8), (64, 1, 4), (32, 2, 2), (64, 1, 1)))
    # of a small layer that costs less than the grouped form's launches
    assert streams(32, 2, 8, 512, 128) and streams(8, 2, 8, 1024, 256)


@pytest.mark.parametrize("E,k,H,I", [(8, 2, 4096, 14336), (8, 2, 128, 8192), (1, 1, 16, 4096), (128, 8, 2816, 704),
                                     (4, 1, 64, 2048), (64, 6, 256, 64), (1024, 32, 512, 1024), (2, 32, 16, 6400)])
def test_workspace_of_more_tokens_serves_fewer(lib, E, k, H, I):
    sizes = [lib.aeoq_moe_fp8_block_workspace_size(T, k, E, H, I) for T in range(300)]
    assert sizes == sorted(sizes)
    for N, K in ((1408, 2816), (40000, 16)):
        sizes = [lib.aeoq_fp8_block_linear_workspace_size(M, N, K) for M in range(300)]
        assert sizes == sorted(sizes)
