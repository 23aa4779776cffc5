"""Both decoders built from models of the library: against its own forward pass in fp32 on the CPU, and what they refuse
because they would compute something else."""
import pytest
import torch

from merak_amd.inference import LlamaDecoder, PagedLlamaDecoder

transformers = pytest.importorskip("transformers")
SIZES = dict(hidden_size=512, intermediate_size=1024, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
             num_hidden_layers=2, vocab_size=1000, max_position_embeddings=128, rms_norm_eps=1e-5, attn_implementation="eager",
             tie_word_embeddings=False)


def build(name, seed=0, **over):
    torch.manual_seed(300 + seed)
    model = getattr(transformers, name + "ForCausalLM")(getattr(transformers, name + "Config")(**{**SIZES, **over})).eval()
    for p in model.parameters():
        if p.dim() == 1:
            p.data.uniform_(0.5, 1.5)
        p.data = p.data.bfloat16().float()              # values a bf16 copy holds exactly
    return model


@pytest.mark.gpu
@pytest.mark.parametrize("name,over", [("Llama", {}), ("Llama", dict(head_dim=64)), ("Qwen3", {}), ("Qwen3", dict(head_dim=64)),
                                       ("Mistral", dict(sliding_window=None))])
def test_paged_decoder_matches_the_library_forward_pass(gpu, name, over):
    """Prompts in two chunks, then single tokens, of two requests.  Two blocks of bf16 roundings: 4e-2 norm-wise, the bound
    of the one-token decoder's test (twice the 2e-2 of a block)."""
    model = build(name, 1, **over)
    if name == "Qwen3":                                 # weights that a decoder without the norms would be far off with
        assert all(layer.self_attn.q_norm.weight.std() > 0.1 for layer in model.model.layers)
    g = torch.Generator().manual_seed(4)
    text = torch.randint(0, 1000, (2, 40), generator=g)
    with torch.no_grad():
        full = model(input_ids=text).logits
    dec = PagedLlamaDecoder.from_hf(model.bfloat16().to(gpu), max_len=64, slots=2, page_size=16)
    at, worst = [0, 0], 0.0
    for step in ([21, 1], [10, 30], *([1, 1],) * 9):
        out = dec.logits(dec.append(torch.cat([text[r, at[r]:at[r] + n] for r, n in enumerate(step)]).to(gpu), step)).float().cpu()
        t0 = 0
        for r, n in enumerate(step):
            want = full[r, at[r]:at[r] + n]
            worst = max(worst, ((out[t0:t0 + n] - want).norm() / want.norm()).item())
            t0 += n
            at[r] += n
    assert at == [40, 40] and dec.lens.tolist() == [40, 40] and worst < 4e-2, worst


def refused(name, match, paged_only=False, change=None, **over):
    model = build(name, 2, **over)
    if change:
        change(model)
    for cls in (PagedLlamaDecoder,) if paged_only else (PagedLlamaDecoder, LlamaDecoder):
        with pytest.raises(ValueError, match=match):
            cls.from_hf(model.bfloat16(), max_len=64)


def test_biases_are_refused():
    refused("Qwen2", "q_proj has a bias")
    refused("Llama", "q_proj has a bias", attention_bias=True)
    refused("Llama", "gate_proj has a bias", mlp_bias=True)
    refused("Llama", "lm_head has a bias", change=lambda m: setattr(m, "lm_head", torch.nn.Linear(512, 1000)))


def test_other_norms_are_refused():
    refused("Gemma", "input_layernorm|activation|norm", hidden_act="silu")              # scales by 1 + weight
    class OnePlus(torch.nn.Module):
        def __init__(self, dim):
            super().__init__()
            self.weight = torch.nn.Parameter(torch.full((dim,), 0.5))

        def forward(self, x):
            y = x.float()
            return ((1 + self.weight.float()) * y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5)).to(x.dtype)

    refused("Qwen3", "layer 1: k_norm is not", True, lambda m: setattr(m.model.layers[1].self_attn, "k_norm", OnePlus(128)))
    refused("Llama", "^[^:]*: norm is not", change=lambda m: setattr(m.model, "norm", OnePlus(512)))
    refused("Llama", "layer 0: input_layernorm is not", change=lambda m: setattr(m.model.layers[0], "input_layernorm",
                                                                                torch.nn.LayerNorm(512, eps=1e-5, bias=False)))
    def other_eps(m):
        m.model.layers[1].self_attn.q_norm.variance_epsilon = 1e-6
    refused("Qwen3", "layer 1: q_norm is not", True, other_eps)


def test_other_arithmetic_is_refused():
    refused("Llama", "activation gelu", hidden_act="gelu")
    refused("Granite", "scores scaled|multiplier|scaling", attention_multiplier=0.5)
    refused("Granite", "residual_multiplier", residual_multiplier=0.3)
    refused("Mistral", "sliding window", sliding_window=32)
    by_kind = {"full_attention": {"rope_theta": 5e5, "rope_type": "default"}}
    refused("Llama", "by kind of layer", change=lambda m: m.config.__dict__.update(rope_parameters=by_kind))
    refused("Qwen3", "sliding window", use_sliding_window=True, sliding_window=32, max_window_layers=1)


def test_head_norms_are_refused_where_there_is_no_place_for_them():
    with pytest.raises(ValueError, match="k_norm, q_norm"):
        LlamaDecoder.from_hf(build("Qwen3", 3).bfloat16(), max_len=64)
