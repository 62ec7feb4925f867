"""LinearFP8Block, Gemma4TextExpertsFP8Block and their loader: layouts on the
CPU; on the GPU conversion, forward, saving and loading, and the routing
with the experts as one layer, against the 64-bit oracle."""
import types

import pytest
import torch
import torch.nn as nn

from oracle import fp8_block as O
from oracle.route_topk import route_topk as route_oracle

F8 = torch.float8_e4m3fn


def config(E=8, H=256, I=192, act="gelu_pytorch_tanh"):
    return types.SimpleNamespace(num_experts=E, hidden_size=H, moe_intermediate_size=I, hidden_activation=act)


def test_layouts_cpu():
    from aeo_quant_b200.bridges.gemma4 import Gemma4TextExpertsFP8Block
    from aeo_quant_b200.bridges.gemma4.linear_fp8 import LinearFP8Block
    m = LinearFP8Block(2816, 2112, bias=True)
    sd = m.state_dict()
    assert set(sd) == {"weight", "weight_scale", "bias"}
    assert sd["weight"].shape == (2112, 2816) and sd["weight"].dtype == F8
    assert sd["weight_scale"].shape == (17, 22) and sd["weight_scale"].dtype == torch.float32
    assert not m.weight.requires_grad and "block=128x128" in repr(m)
    with pytest.raises(ValueError, match="multiple of 16"):
        LinearFP8Block(100, 64)
    e = Gemma4TextExpertsFP8Block(config())
    sd = e.state_dict()
    assert sd["gate_up_proj"].shape == (8, 384, 256) and sd["gate_up_proj_scale"].shape == (8, 3, 2)
    assert sd["down_proj"].shape == (8, 256, 192) and sd["down_proj_scale"].shape == (8, 2, 2)
    assert sd["down_proj"].dtype == F8 and sd["down_proj_scale"].dtype == torch.float32
    with pytest.raises(ValueError, match="hidden_activation"):
        Gemma4TextExpertsFP8Block(config(act="relu"))


def test_class_swap_and_dispatch_cpu(monkeypatch):
    from transformers.models.gemma4 import modeling_gemma4 as G
    from aeo_quant_b200.bridges.gemma4 import loader
    from aeo_quant_b200.bridges.gemma4.modeling_fp8_block import Gemma4TextExpertsFP8Block
    before = G.Gemma4TextExperts
    with pytest.raises(RuntimeError):
        with loader.gemma4_experts_fp8_block_class_swap():
            assert G.Gemma4TextExperts is Gemma4TextExpertsFP8Block
            raise RuntimeError
    assert G.Gemma4TextExperts is before
    seen = []
    monkeypatch.setattr(loader, "load_gemma4_fp8_block", lambda path, **kw: seen.append((path, kw)))
    loader.load_gemma4("p", quant_format="fp8_block", device_map="cpu")
    assert seen == [("p", {"device_map": "cpu"})]


@pytest.mark.parametrize("act", ["gelu_pytorch_tanh", "silu", "relu"])
def test_conversion_keeps_the_activation_cpu(monkeypatch, act):
    """Experts are converted with the activation they have, or refused before
    any of them is replaced."""
    from transformers.models.gemma4.modeling_gemma4 import Gemma4TextExperts
    from aeo_quant_b200.bridges.gemma4 import loader
    from aeo_quant_b200.bridges.gemma4.modeling_fp8_block import Gemma4TextExpertsFP8Block
    from aeo_quant_b200.gpu import quant
    monkeypatch.setattr(quant, "quantize_3d_to_fp8_block", lambda w: (
        w.to(F8), torch.ones(w.shape[0], -(-w.shape[1] // 128), -(-w.shape[2] // 128))))
    model = nn.Module()
    model.experts = Gemma4TextExperts(config(act=act))
    for p in model.experts.parameters():
        nn.init.zeros_(p)
    if act == "relu":
        with pytest.raises(ValueError, match="not supported"):
            loader.quantize_experts_to_fp8_block(model)
        assert type(model.experts) is Gemma4TextExperts
        return
    assert loader.quantize_experts_to_fp8_block(model) == 1
    assert type(model.experts) is Gemma4TextExpertsFP8Block
    assert model.experts.activation == act and model.experts.gate_up_proj_scale.shape == (8, 3, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,N,K,bias", [((7,), 2112, 2816, False), ((2, 5), 200, 144, True), ((1,), 96, 64, True),
                                            ((3, 50), 384, 256, False)])
def test_linear_module(shape, N, K, bias):
    from aeo_quant_b200.bridges.gemma4.linear_fp8 import LinearFP8Block
    torch.manual_seed(N)
    lin = nn.Linear(K, N, bias=bias).to(device="cuda", dtype=torch.bfloat16)
    m = LinearFP8Block.from_linear(lin)
    rq, rs = O.quantize_blocks(lin.weight.detach().double()[None])
    assert torch.equal(m.weight.double(), rq[0]) and torch.equal(m.weight_scale.double(), rs[0])
    x = torch.randn(*shape, K, device="cuda").to(torch.bfloat16)
    y = m(x)
    ref, tol = O.linear(x.reshape(-1, K).double(), rq[0], rs[0], lin.bias.detach().double() if bias else None)
    assert y.shape == (*shape, N) and bool(((y.reshape(-1, N).double() - ref).abs() <= tol).all())
    back = LinearFP8Block(K, N, bias=bias, device="cuda")
    back.load_state_dict(m.state_dict())
    assert torch.equal(back(x), y)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 33, 300])
def test_routing_and_experts_together(T):
    """Logits to layer output: sigmoid scores, balance bias and groups choose
    the experts, whose block-scaled MLPs are summed with the routing weights."""
    from aeo_quant_b200.bridges.gemma4.modeling_fp8_block import Gemma4TextExpertsFP8Block
    from aeo_quant_b200.gpu.quant import quantize_3d_to_fp8_block
    from aeo_quant_b200.gpu.routing import route_topk
    E, H, I, k = 32, 512, 192, 4
    g = torch.Generator(device="cuda").manual_seed(T)
    m = Gemma4TextExpertsFP8Block(config(E, H, I, "silu")).cuda()
    for name in ("gate_up_proj", "down_proj"):
        q, s = quantize_3d_to_fp8_block(torch.randn(getattr(m, name).shape, generator=g, device="cuda") * 0.05)
        getattr(m, name).data.copy_(q)
        getattr(m, f"{name}_scale").copy_(s)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    gate = torch.randn(E, H, generator=g, device="cuda") * 0.05
    bias = torch.randn(E, generator=g, device="cuda") * 0.1
    logits = x.float() @ gate.T
    logits[:, 5] = float("-inf")                   # an expert that is switched off
    kw = dict(score="sigmoid", n_group=4, topk_group=2, group_score="top2", scale=2.5)
    w, ids = route_topk(logits, k, bias=bias, **kw)
    y = m(x, ids, w)
    rw, ri = route_oracle(logits.double().cpu().numpy(), k, bias=bias.double().cpu().numpy(), **kw)
    assert (ids.cpu().numpy() == ri).all() and 5 not in ri
    ref, tol = O.experts(x.double(), ids, torch.from_numpy(rw).cuda(), m.gate_up_proj.double(),
                         m.gate_up_proj_scale.double(), m.down_proj.double(), m.down_proj_scale.double(), "silu")
    tol = tol + 8e-6 * ref.abs().amax(1, keepdim=True) * k       # the weights' own f32 error
    assert bool(((y.double() - ref).abs() <= tol).all())
    # the same as one captured graph
    bx, bl = torch.zeros_like(x), torch.zeros_like(logits)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w2, i2 = route_topk(bl, k, bias=bias, **kw)
        out = m(bx, i2, w2)
    bx.copy_(x)
    bl.copy_(logits)
    graph.replay()
    assert torch.equal(out, y) and torch.equal(i2, ids)


@pytest.mark.gpu
def test_stack_converted_saved_and_loaded(tmp_path):
    """A small random-init Gemma-4 decoder with its experts converted on the
    GPU: the saved checkpoint loads under the class swap and generates the
    same greedy tokens; each layer's experts agree with the oracle."""
    from test_stack_gpu import small_config
    from transformers.models.gemma4.modeling_gemma4 import Gemma4ForCausalLM
    from aeo_quant_b200.bridges.gemma4.loader import load_gemma4, quantize_experts_to_fp8_block, swap_routers
    from aeo_quant_b200.bridges.gemma4.modeling_fp8_block import Gemma4TextExpertsFP8Block
    torch.manual_seed(0)
    model = Gemma4ForCausalLM(small_config()).to(device="cuda", dtype=torch.bfloat16).eval()
    for layer in model.model.layers:
        nn.init.normal_(layer.router.proj.weight, std=0.5)
    ids = torch.randint(10, 4096, (1, 40), generator=torch.Generator().manual_seed(3)).cuda()
    assert quantize_experts_to_fp8_block(model) == 2
    assert all(isinstance(l.experts, Gemma4TextExpertsFP8Block) for l in model.model.layers)
    assert quantize_experts_to_fp8_block(model) == 0
    model.save_pretrained(tmp_path / "out")
    swap_routers(model)
    loaded = load_gemma4(str(tmp_path / "out"), quant_format="fp8_block", device_map="cuda").eval()
    assert loaded.model.layers[0].experts.gate_up_proj.dtype == F8
    assert loaded.model.layers[0].experts.down_proj_scale.dtype == torch.float32
    with torch.no_grad():
        a = loaded.generate(ids, max_new_tokens=6, min_new_tokens=6, do_sample=False)
        b = model.generate(ids, max_new_tokens=6, min_new_tokens=6, do_sample=False)
    assert torch.equal(a, b)
    for layer in model.model.layers:                 # the layer's forward against the oracle, prefill and one token
        e = layer.experts
        for T in (1, 40):
            x = torch.randn(T, 512, device="cuda").to(torch.bfloat16)
            with torch.no_grad():
                _, w, i = layer.router(x)
                y = e(x, i, w)
            ref, tol = O.experts(x.double(), i, w.double(), e.gate_up_proj.double(), e.gate_up_proj_scale.double(),
                                 e.down_proj.double(), e.down_proj_scale.double(), "gelu_pytorch_tanh")
            assert bool(((y.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("bad", [dict(H=264), dict(I=96), dict(E=1025, H=16, I=64)])
def test_sizes_that_the_kernels_do_not_take_are_refused_cpu(monkeypatch, bad):
    """By the module, and by the conversion before any layer is replaced."""
    from transformers.models.gemma4.modeling_gemma4 import Gemma4TextExperts
    from aeo_quant_b200.bridges.gemma4 import Gemma4TextExpertsFP8Block, loader
    from aeo_quant_b200.gpu import quant
    with pytest.raises(ValueError, match="multiple of 16"):
        Gemma4TextExpertsFP8Block(config(**bad))
    monkeypatch.setattr(quant, "quantize_3d_to_fp8_block", lambda w: (
        w.to(F8), torch.ones(w.shape[0], -(-w.shape[1] // 128), -(-w.shape[2] // 128))))
    model = nn.Module()
    model.good, model.bad = Gemma4TextExperts(config()), Gemma4TextExperts(config(**bad))
    for p in model.parameters():
        nn.init.zeros_(p)
    with pytest.raises(ValueError, match="multiple of 16"):
        loader.quantize_experts_to_fp8_block(model)
    assert type(model.good) is Gemma4TextExperts and type(model.bad) is Gemma4TextExperts
    del model.bad
    assert loader.quantize_experts_to_fp8_block(model) == 1 and type(model.good) is Gemma4TextExpertsFP8Block
