"""The paged-cache operators run together as a decoder runs them: against the one-token decoder of this package, against a
causal forward pass in fp32, and speculative steps against plain greedy ones."""
import pytest
import torch
import torch.nn.functional as F

from merak_amd import ops
from merak_amd.inference import LlamaDecoder, PagedLlamaDecoder, rope_tables
from merak_amd.inference.llama_decode import LlamaBlockWeights
from oracle import tp_reference as R

pytestmark = pytest.mark.gpu
H, I, V, NQ, NKV, D, LAYERS = 512, 1024, 1000, 4, 2, 128, 2


def model(gpu, seed=0, head_dim=D):
    g = torch.Generator().manual_seed(100 + seed)
    mk = lambda *s: (torch.randn(*s, generator=g) * 0.05).bfloat16()
    ones = lambda n: (torch.rand(n, generator=g) * 0.2 + 0.9).bfloat16()
    blocks = [LlamaBlockWeights(ones(H), mk((NQ + 2 * NKV) * head_dim, H), mk(H, NQ * head_dim), ones(H), mk(2 * I, H), mk(H, I))
              for _ in range(LAYERS)]
    embed, final, head = (torch.randn(V, H, generator=g)).bfloat16(), ones(H), mk(V, H) * 4
    return embed, blocks, final, head


def on(gpu, m):
    embed, blocks, final, head = m
    mv = lambda b: LlamaBlockWeights(*[getattr(b, f).to(gpu) for f in ("input_norm", "qkv", "o", "post_norm", "gate_up", "down")])
    return embed.to(gpu), [mv(b) for b in blocks], final.to(gpu), head.to(gpu)


def forward_fp32(m, tokens, norms=None, head_dim=D):
    """Hidden states of all positions of one sequence, fp32 on the CPU."""
    embed, blocks, final, _ = m
    n = len(tokens)
    x, res = embed.float()[tokens], None
    cos, sin = rope_tables(head_dim, n, 10000.0)
    for i, w in enumerate(blocks):
        h, res = R.rms_norm(x, w.input_norm.float(), 1e-5, res)
        qkv = F.linear(h, w.qkv.float()).view(n, NQ + 2 * NKV, head_dim)
        q, k, v = qkv[:, :NQ], qkv[:, NQ:NQ + NKV], qkv[:, NQ + NKV:]
        if norms is not None:
            q = R.rms_norm(q, norms[0][i].float(), 1e-5)[0]
            k = R.rms_norm(k, norms[1][i].float(), 1e-5)[0]
        q, k = R.apply_rope(q, cos, sin), R.apply_rope(k, cos, sin)
        k, v = k.repeat_interleave(NQ // NKV, 1), v.repeat_interleave(NQ // NKV, 1)
        s = torch.einsum("ihd,jhd->hij", q, k) * head_dim ** -0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), float("-inf")).softmax(-1)
        o = F.linear(torch.einsum("hij,jhd->ihd", s, v).reshape(n, -1), w.o.float())
        h, res = R.rms_norm(o, w.post_norm.float(), 1e-5, res)
        x = F.linear(R.swiglu(F.linear(h, w.gate_up.float())), w.down.float())
    return R.rms_norm(x, final.float(), 1e-5, res)[0]


def rel(a, b):
    a, b = a.double().cpu(), b.double()
    return ((a - b).norm() / b.norm()).item()


@pytest.mark.parametrize("head_dim,norms", [(128, False), (64, True)])
def test_prompts_in_chunks_and_single_tokens_against_a_causal_pass(gpu, head_dim, norms):
    """Three requests of different lengths, their prompts in uneven chunks mixed with single tokens of others; a fourth
    slot never used, one released and used again.  bf16 activations between fp32 sums: 2e-2 norm-wise, as for the
    one-token decoder's block."""
    m = model(gpu, 1, head_dim)
    g = torch.Generator().manual_seed(5)
    nw = None
    if norms:
        nw = [[(torch.rand(head_dim, generator=g) + 0.5).bfloat16() for _ in range(LAYERS)] for _ in range(2)]
    embed, blocks, final, head = on(gpu, m)
    dec = PagedLlamaDecoder(embed, blocks, final, head, NQ, NKV, head_dim, max_len=256, slots=4, page_size=16, n_pages=30,
                            q_norms=[w.to(gpu) for w in nw[0]] if norms else None,
                            k_norms=[w.to(gpu) for w in nw[1]] if norms else None)
    text = [torch.randint(0, V, (n,), generator=g) for n in (150, 37, 90)]
    rows = [forward_fp32(m, t, nw, head_dim) for t in text]
    at = [0, 0, 0]
    for step in ([100, 1, 0], [1, 20, 64], [33, 1, 1], [0, 15, 25], [16, 0, 0]):
        toks = torch.cat([text[r][at[r]:at[r] + n] for r, n in enumerate(step)])
        out = dec.append(toks.to(gpu), step + [0])
        assert dec.granted.all()
        t0 = 0
        for r, n in enumerate(step):
            if n:
                assert rel(out[t0:t0 + n], rows[r][at[r]:at[r] + n]) < 2e-2, (step, r)
            t0 += n
            at[r] += n
    assert dec.lens.tolist() == [150, 37, 90, 0] and dec.free_count.item() == 30 - 10 - 3 - 6
    # a request too large for the pool is refused and leaves the others alone
    dec.append(torch.zeros(200, dtype=torch.int64, device=gpu), [0, 0, 0, 200])
    assert dec.granted.tolist() == [True, True, True, False] and dec.lens[3].item() == 0 and dec.free_count.item() == 11
    dec.release([0, 2])
    assert dec.free_count.item() == 27 and dec.lens.tolist() == [0, 37, 0, 0]
    out = dec.append(text[2][:50].to(gpu), [0, 0, 0, 50])
    assert rel(out, rows[2][:50]) < 2e-2


def test_greedy_steps_match_the_one_token_decoder(gpu):
    """Logits of the two decoders for the same text (bf16 roundings in different places: 2e-2 norm-wise), single tokens."""
    embed, blocks, final, head = on(gpu, model(gpu, 2))
    one = LlamaDecoder(embed, blocks, final, head, NQ, NKV, D, max_len=64, batch=2)
    paged = PagedLlamaDecoder(embed, blocks, final, head, NQ, NKV, D, max_len=64, slots=2, page_size=16)
    tok = torch.tensor([3, 700], device=gpu)
    for _ in range(40):
        a, b = one.logits(tok), paged.logits(paged.append(tok, [1, 1]))
        assert rel(b, a.double().cpu()) < 2e-2
        tok = a.argmax(-1)
    nxt = paged.step(tok[:1], [1, 0])
    assert nxt[1].item() == -1 and 0 <= nxt[0].item() < V


def test_speculative_steps_keep_what_the_target_would_have_said(gpu):
    """top_k = 1 makes the target certain: drafts that are its own greedy continuation are all accepted, wrong ones are
    cut off at the first mistake and the drawn token is the greedy one; the cache then holds exactly the kept tokens."""
    m = on(gpu, model(gpu, 3))
    mk = lambda: PagedLlamaDecoder(m[0], m[1], m[2], m[3], NQ, NKV, D, max_len=128, slots=2, page_size=16)
    plain, spec = mk(), mk()
    prompt = torch.randint(0, V, (2, 21), generator=torch.Generator().manual_seed(1)).to(gpu)
    # teacher: greedy tokens from the same kernels, one step of many tokens, so that near ties cannot fall differently
    tok = plain.step(prompt.reshape(-1), [21, 21])
    spec.append(prompt.reshape(-1), [21, 21])
    last, kept = tok.clone(), [[], []]
    g = torch.Generator().manual_seed(2)
    for k in range(6):
        K = 3
        start = spec.lens.clone()
        # drafts: for the first request what the target says for them (found by running them), for the second noise
        drafts = torch.randint(0, V, (2, K), generator=g).to(gpu)
        probe = mk()
        probe.append(prompt.reshape(-1), [21, 21])
        if kept[0] or kept[1]:
            probe.append(torch.tensor(kept[0] + kept[1], device=gpu), [len(kept[0]), len(kept[1])])
        cur = last.clone()
        for i in range(K):
            cur = probe.step(cur, [1, 1])
            drafts[0, i] = cur[0]
            cur[1] = drafts[1, i]
        tokens, n = spec.verify(last, drafts, torch.rand(2, K + 1, generator=g).to(gpu), top_k=1)
        assert tokens.shape == (2, K + 1) and 0 <= n[1].item() <= K
        for r in range(2):
            a = n[r].item()
            assert torch.equal(tokens[r, :a], drafts[r, :a]) and 0 <= tokens[r, a].item() < V
            assert (tokens[r, a + 1:] == -1).all()
            assert spec.lens[r].item() == start[r].item() + 1 + a
            kept[r] += [last[r].item()] + drafts[r, :a].tolist()
            last[r] = tokens[r, a]
        # the cache holds the kept tokens and nothing else: the next hidden row is that of a fresh decoder
        check = mk()
        check.append(prompt.reshape(-1), [21, 21])
        check.append(torch.tensor(kept[0] + kept[1], device=gpu), [len(kept[0]), len(kept[1])])
        assert check.lens.tolist() == spec.lens.tolist()
        held, free, lens = spec.held, spec.free_count, spec.lens
        a, b = spec.append(last, [1, 1]), check.append(last, [1, 1])
        assert rel(a, b.double().cpu()) < 2e-2
        spec.lens = lens                                     # the probe token leaves again
    assert len(kept[0]) > len(kept[1])
