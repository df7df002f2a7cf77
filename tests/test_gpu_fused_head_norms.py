"""Decoders with per-head q/k norms under fuse_llama: calls that the fused forwards have to leave to the
modules, and what they must not touch."""
import copy

import pytest
import torch
import torch.nn as nn

from test_gpu_distill import model_with_head_norms

pytestmark = pytest.mark.gpu


def hidden(seed=1, dtype=torch.bfloat16, shape=(2, 24, 256)):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def pair(dtype=torch.bfloat16, seed=0):
    """The same small model twice, the second with the fused forwards; eager attention, which torch
    can differentiate forward."""
    from zotitan_b200.llama_fused import fuse_llama
    m = model_with_head_norms(seed=seed, layers=1).to(dtype)
    m.config._attn_implementation = "eager"
    f = copy.deepcopy(m)
    fuse_llama(f)
    return m, f


def tables(m, x):
    return m.model.rotary_emb(x, torch.arange(x.shape[1], device="cuda")[None])


PARTS = {"norm": lambda m, x, pe: m.model.norm(x), "attention": lambda m, x, pe: m.model.layers[0].self_attn(x, pe, None)[0],
         "mlp": lambda m, x, pe: m.model.layers[0].mlp(x)}


@pytest.mark.parametrize("no_grad", [True, False])
@pytest.mark.parametrize("part", PARTS)
def test_forward_mode(part, no_grad):
    """Forward-mode derivatives, which torch.no_grad leaves on: those of the modules."""
    import torch.autograd.forward_ad as fw
    m, f = pair()
    x, t = hidden(1), hidden(2)
    pe = tables(m, x)
    out = []
    for model in (m, f):
        for p in model.parameters():
            p.requires_grad_(False)
        with torch.set_grad_enabled(not no_grad), fw.dual_level():
            out.append(fw.unpack_dual(PARTS[part](model, fw.make_dual(x, t), pe)))
    assert torch.equal(out[0].primal, out[1].primal)
    assert out[1].tangent is not None and torch.equal(out[0].tangent, out[1].tangent)


def test_forward_mode_in_a_weight():
    """A tangent on a norm's weight alone, reached through the head norms and the decoder norm."""
    import torch.autograd.forward_ad as fw
    m, f = pair()
    x = hidden(3)
    pe = tables(m, x)
    for part, name in (("attention", "model.layers.0.self_attn.q_norm"), ("norm", "model.norm")):
        out = []
        for model in (m, f):
            mod = model.get_submodule(name)
            w = mod.weight.detach()
            with torch.no_grad(), fw.dual_level():
                mod.weight = nn.Parameter(w, requires_grad=False)
                del mod._parameters["weight"]
                mod.weight = fw.make_dual(w, torch.ones_like(w))
                out.append(fw.unpack_dual(PARTS[part](model, x, pe)).tangent.clone())
                del mod.weight
                mod.weight = nn.Parameter(w, requires_grad=False)
        assert torch.equal(out[0], out[1]) and bool(out[1].any())


@pytest.mark.parametrize("part", PARTS)
def test_traced(part):
    """A trace holds the modules' operations, so it computes on other inputs too."""
    m, f = pair()
    x, other = hidden(4), hidden(5)
    pe = tables(m, x)
    for p in f.parameters():
        p.requires_grad_(False)
    with torch.no_grad():
        traced = torch.jit.trace(lambda h: PARTS[part](f, h, pe), x, check_trace=False)
        want = PARTS[part](m, other, pe)
        assert torch.equal(traced(other), want)


@pytest.mark.parametrize("part", PARTS)
def test_function_transforms(part):
    """torch.func's gradient and vmap over a fused module: those over the module."""
    m, f = pair(torch.float32 if part == "attention" else torch.bfloat16)
    x = hidden(6, m.dtype)
    pe = tables(m, x)
    got, want = (torch.func.grad(lambda h: PARTS[part](model, h, pe).float().square().sum())(x) for model in (f, m))
    assert torch.equal(got, want)
    with torch.no_grad():
        both = torch.stack([x, -x])
        got, want = (torch.func.vmap(lambda h: PARTS[part](model, h, pe))(both) for model in (f, m))
    assert torch.equal(got, want)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("part", PARTS)
def test_compiled_whole(part, grad):
    """torch.compile without graph breaks, as over the modules."""
    m, f = pair()
    x = hidden(7)
    pe = tables(m, x)
    torch._dynamo.reset()
    with torch.set_grad_enabled(grad):
        got = torch.compile(lambda h: PARTS[part](f, h, pe), fullgraph=True, backend="eager")(x)
        assert torch.equal(got, PARTS[part](m, x, pe))
    torch._dynamo.reset()


def test_trainable_frequencies():
    """A rotary embedding whose frequencies are trained: the gradient of cos and sin is the modules'."""
    m, f = pair(torch.float32)
    x = hidden(8, torch.float32)
    grads = []
    for model in (m, f):
        freq = model.model.rotary_emb.inv_freq.detach().clone().requires_grad_()
        ang = torch.arange(x.shape[1], device="cuda")[:, None] * freq
        ang = torch.cat((ang, ang), -1)[None]
        out = model.model.layers[0].self_attn(x, (ang.cos(), ang.sin()), None)[0]
        grads.append(torch.autograd.grad(out.square().sum(), freq)[0])
    assert torch.equal(*grads) and bool(grads[0].any())
    with torch.no_grad():     # the same tables in an evaluation
        outs = [model.model.layers[0].self_attn(x, (ang.cos().requires_grad_(), ang.sin().requires_grad_()), None)[0] for model in (m, f)]
    assert torch.equal(*outs)


class Keep(nn.Module):
    """A projection that hands out a tensor it goes on holding."""

    def __init__(self, out):
        super().__init__()
        self.out = out

    def forward(self, x):
        return self.out


def llama_attention():
    from transformers import LlamaConfig, LlamaForCausalLM
    from zotitan_b200.llama_fused import fuse_llama
    cfg = LlamaConfig(vocab_size=100, hidden_size=256, intermediate_size=512, num_hidden_layers=1, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=64, attn_implementation="sdpa")
    torch.manual_seed(0)
    m = LlamaForCausalLM(cfg).to("cuda", torch.bfloat16).eval()
    fuse_llama(m)
    return m


@pytest.mark.parametrize("how", ["hook", "every_module_hook", "adapter_hook", "base_hook", "module"])
@pytest.mark.parametrize("llama", [False, True])
def test_projection_outputs_that_others_hold(how, llama):
    """What a hook took from a projection, or a projection holds itself, stays as it was."""
    from zotitan_b200.lora import LoRALinear
    f = llama_attention() if llama else pair()[1]
    x = hidden(9)
    pe = tables(f, x)
    attn = f.model.layers[0].self_attn
    if "hook" in how and how.split("_")[0] in ("adapter", "base"):
        for name in ("q_proj", "k_proj"):
            setattr(attn, name, LoRALinear(getattr(attn, name), 8, 16).cuda())
    with torch.inference_mode():
        q, k = attn.q_proj(x), attn.k_proj(x)
        want = attn(x, pe, None)[0]
        seen = {}
        handles = []
        if how in ("hook", "adapter_hook", "base_hook"):
            for name in ("q_proj", "k_proj"):
                mod = getattr(attn, name)
                if how == "base_hook":
                    mod.lora_A.weight.zero_()     # lora_B is zero: nothing is added to what the base gives out
                    mod = mod.base_linear
                handles.append(mod.register_forward_hook(lambda mod, a, out, name=name: seen.__setitem__(name, out)))
        elif how == "every_module_hook":
            names = {attn.q_proj: "q_proj", attn.k_proj: "k_proj"}
            handles.append(nn.modules.module.register_module_forward_hook(
                lambda mod, a, out: seen.__setitem__(names[mod], out) if mod in names else None))
        else:
            seen = {"q_proj": q.clone(), "k_proj": k.clone()}
            attn.q_proj, attn.k_proj = Keep(seen["q_proj"]), Keep(seen["k_proj"])
        got = attn(x, pe, None)[0]
        for h in handles:
            h.remove()
    assert torch.equal(seen["q_proj"], q) and torch.equal(seen["k_proj"], k)
    if llama or how != "every_module_hook":     # the hook for every module is also the norms': those run themselves
        assert torch.equal(got, want)


def test_projections_that_share_memory():
    """Query and key heads that a projection gives out as the same memory, or one head for all."""
    m, f = pair()
    x = hidden(10)
    pe = tables(m, x)
    q = hidden(11, shape=(2, 24, 384))
    one = hidden(12, shape=(2, 24, 64))
    for key in (q[..., :128], one.unsqueeze(2).expand(-1, -1, 2, -1)):
        out = []
        with torch.no_grad():
            for model in (m, f):
                attn = model.model.layers[0].self_attn
                attn.q_proj, attn.k_proj = Keep(q.clone()), Keep(None)
                attn.k_proj.out = attn.q_proj.out[..., :128] if key.dim() == 3 else key
                out.append(attn(x, pe, None)[0].float())
        scale = float(out[0].square().mean().sqrt())     # as in test_gpu_distill.test_attention_with_head_norms
        assert float((out[0] - out[1]).square().mean().sqrt()) <= 0.02 * scale


@pytest.mark.parametrize("llama", [False, True])
def test_hooked_projections_of_the_mlp_run(llama):
    """Hooks on gate, up and the activation see their calls, at the sizes of the fused GEMM too."""
    from zotitan_b200.llama_fused import fuse_llama
    m, f = pair()
    mlp = f.model.layers[0].mlp
    if llama:
        from transformers import LlamaConfig
        from transformers.models.llama.modeling_llama import LlamaMLP
        mlp = LlamaMLP(LlamaConfig(hidden_size=256, intermediate_size=512)).to("cuda", torch.bfloat16)
        fuse_llama(mlp)
    x = hidden(13, shape=(2, 128, 256))
    with torch.no_grad():
        want = mlp(x)
        seen = []
        for mod in (mlp.gate_proj, mlp.up_proj, mlp.act_fn):
            h = mod.register_forward_hook(lambda mod, a, out: seen.append(mod))
            got = mlp(x)
            h.remove()
            assert seen == [mod]
            seen.clear()
            assert float((got - want).float().square().mean().sqrt()) <= 0.01 * float(want.float().square().mean().sqrt())
        h = mlp.gate_proj.register_forward_hook(lambda mod, a, out: out * 0)
        assert not mlp(x).any()
        h.remove()


def test_hooks_for_every_module_reach_the_head_norms():
    m, f = pair()
    x = hidden(14)
    pe = tables(m, x)
    attn = f.model.layers[0].self_attn
    seen = []
    h = nn.modules.module.register_module_forward_hook(lambda mod, a, out: seen.append(mod))
    with torch.no_grad():
        got = attn(x, pe, None)[0]
    h.remove()
    assert attn.q_norm in seen and attn.k_norm in seen
    with torch.no_grad():
        want = m.model.layers[0].self_attn(x, pe, None)[0]
    scale = float(want.float().square().mean().sqrt())
    assert float((got - want).float().square().mean().sqrt()) <= 0.02 * scale


class InFp32(nn.Module):
    def __init__(self, base):
        super().__init__()
        self.base = base

    def forward(self, x):
        return nn.functional.linear(x.float(), self.base.weight.float())


@pytest.mark.parametrize("grad", [False, True])
def test_projections_in_another_type(grad):
    """Projections that answer in fp32 to bf16 hidden states: the head norms run as modules there."""
    m, f = pair()
    x = hidden(15)
    pe = tables(m, x)
    out = []
    for model in (m, f):
        attn = model.model.layers[0].self_attn
        for name in ("q_proj", "k_proj", "v_proj", "o_proj"):
            setattr(attn, name, InFp32(getattr(attn, name)))
        with torch.set_grad_enabled(grad):
            out.append(attn(x, pe, None)[0])
    assert out[0].dtype == torch.float32 and torch.equal(*out)


def test_replaced_forwards_are_called():
    """A forward set on an instance, as offloading and kernel hubs do: before or after fuse_llama, on a norm, a
    projection or the activation."""
    from zotitan_b200.llama_fused import fuse_llama, unfuse_llama
    x = hidden(16, shape=(2, 128, 256))
    where = {"attention": ("q_norm", "k_norm", "q_proj"), "mlp": ("gate_proj", "up_proj", "act_fn"), "norm": ("",)}
    for part, names in where.items():
        for name in names:
            for before in (True, False):
                m, f = pair()
                pe = tables(m, x)
                out = []
                for model in (m, f):
                    root = {"attention": model.model.layers[0].self_attn, "mlp": model.model.layers[0].mlp, "norm": model.model.norm}[part]
                    mod = root.get_submodule(name)
                    if before:
                        unfuse_llama(model)
                    own = mod.forward
                    mod.forward = lambda h, own=own: own(h) * 2
                    if before and model is f:
                        fuse_llama(model)
                    with torch.no_grad():
                        out.append(PARTS[part](model, x, pe).float())
                scale = float(out[0].square().mean().sqrt())
                assert float((out[0] - out[1]).square().mean().sqrt()) <= 0.02 * scale, (part, name, before)


def test_compiled_llama():
    """A fused Llama under torch.compile: its modules' own code, as compiled without fuse_llama."""
    from zotitan_b200.llama_fused import unfuse_llama
    m = llama_attention()
    ids = torch.arange(40, device="cuda").view(2, 20) % 100
    torch._dynamo.reset()
    with torch.inference_mode():
        got = torch.compile(lambda i: m(input_ids=i, use_cache=False).logits, backend="eager")(ids)
        unfuse_llama(m)
        assert torch.equal(got, m(input_ids=ids, use_cache=False).logits)
    torch._dynamo.reset()
