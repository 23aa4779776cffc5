"""The paged-cache operators captured into graphs that are replayed with other inputs, on two streams at once, and the
decoder in half precision and with many slots."""
import pytest
import torch

from merak_amd import mpu, ops
from merak_amd.inference import PagedLlamaDecoder
from merak_amd.inference.llama_decode import LlamaBlockWeights
from test_paged_decode import D, LAYERS, NKV, NQ, V, forward_fp32, model, on, rel
from test_paged_ops import attn_inputs, check_attn, rotary_case, verify_case

pytestmark = pytest.mark.gpu


def replayed(run, inputs, variants):
    """run() captured once over ``inputs`` (tensors that are overwritten), replayed for every variant (twice, with eager
    work and a synchronisation between) and compared with what it gives eagerly."""
    def load(v):
        for t, s in zip(inputs, v):
            t.copy_(s)

    wants = []
    for v in variants:
        load(v)
        wants.append([t.clone() for t in run()])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for v, want in [*zip(variants, wants)] * 2:
        load(v)
        graph.replay()
        junk = torch.randn(5000, device=inputs[0].device).sum().item()
        assert junk == junk
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_rotary_forward_and_backward_in_a_graph(gpu):
    T, hq, hk, d = 133, 8, 2, 128
    make = lambda seed: [t.to(gpu) for t in rotary_case(T, hq, hk, d, torch.bfloat16, "both", seed)]
    ups = lambda seed: [torch.randn(T, n, d, generator=torch.Generator().manual_seed(seed)).bfloat16().to(gpu) for n in (hq, hk, hk)]
    qkv, cos, sin, pos, qw, kw = make(40)
    up = ups(1)

    def run():
        return [*ops.qk_norm_rope(qkv, cos, sin, pos, hq, qw, kw), *ops.qk_norm_rope_bwd(*up, qkv, cos, sin, pos, qw, kw)]

    variants = []
    for seed in (40, 42, 44):
        a = make(seed)
        variants.append([a[0], a[3], a[4], a[5], *ups(seed)])
    replayed(run, [qkv, pos, qw, kw, *up], variants)


def test_module_form_forward_and_backward_in_a_graph(gpu):
    """Autograd's backward captured too, with no eager graph of the same leaves alive."""
    T, hq, hk, d = 40, 4, 2, 64
    src = [[t.to(gpu) for t in rotary_case(T, hq, hk, d, torch.bfloat16, "both", seed)] for seed in (50, 52, 54)]
    cos, sin = src[0][1], src[0][2]
    qkv, pos, qw, kw = (src[0][i].clone() for i in (0, 3, 4, 5))
    leaves = [t.requires_grad_(True) for t in (qkv, qw, kw)]

    def run():
        q, k, v = mpu.qk_norm_rotary(qkv, cos, sin, pos, hq, qw, kw)
        grads = torch.autograd.grad([q, k, v], leaves, [q.detach(), k.detach(), v.detach()])
        return [q.detach(), k.detach(), v.detach(), *grads]

    with torch.no_grad():
        bufs = [qkv.detach(), pos, qw.detach(), kw.detach()]
    variants = [[s[0], s[3], s[4], s[5]] for s in src]
    side = torch.cuda.Stream(gpu)                       # the warm-up that capturing a backward pass asks for
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream(gpu).wait_stream(side)
    replayed(run, bufs, variants)


@pytest.mark.parametrize("with_draft", [True, False])
def test_verify_draft_in_a_graph(gpu, with_draft):
    cases = [verify_case(5, 3, 20001, torch.float32, with_draft, seed) for seed in (1, 2, 3)]
    variants = [[t.to(gpu) for t in c if t is not None] for c in cases]
    bufs = [t.clone() for t in variants[0]]
    args = (bufs[0], bufs[1], bufs[2] if with_draft else None, bufs[-1])
    replayed(lambda: ops.verify_draft(*args), bufs, variants)


def test_plan_and_release_in_a_graph(gpu):
    """A step that plans, then gives the pages of some requests back, in one graph; the state is part of the inputs."""
    R, cols, page = 7, 6, 16
    g = torch.Generator().manual_seed(3)
    def state(seed):
        lens = torch.randint(0, 60, (R,), generator=g)
        held = ((lens + page - 1) // page).int()
        ids = torch.randperm(R * cols, generator=g).int()
        table, free = torch.full((R, cols), -1, dtype=torch.int32), torch.full((R * cols,), -1, dtype=torch.int32)
        at = 0
        for r, h in enumerate(held.tolist()):
            table[r, :h] = ids[at:at + h]
            at += h
        free[:R * cols - at] = ids[at:]
        new = torch.randint(0, 20, (R,), generator=g)
        done = torch.randint(0, 2, (R,), generator=g).bool()
        return [t.to(gpu) for t in (lens, new, held, table, free, torch.tensor([R * cols - at], dtype=torch.int32), done)]

    variants = [state(i) for i in range(3)]
    lens, new, held, table, free, count, done = bufs = [t.clone() for t in variants[0]]

    def run():
        plan = ops.paged_plan(lens, new, held, table, free, count, page, 150)
        ops.paged_release(done, plan.held, table, free, plan.free_count)
        return [*plan, table, free]

    replayed(run, bufs, variants)


def test_attention_without_a_workspace_of_the_callers_in_two_graphs(gpu):
    """Each capture has a workspace of its own when none is given: two graphs replayed on two streams at once."""
    one = attn_inputs(3, [900, 30, 4000], [1, 1, 1], 32, 8, 128, 16, torch.bfloat16, 70)
    two = attn_inputs(2, [100, 700], [90, 33], 8, 2, 128, 64, torch.bfloat16, 71)
    graphs, outs, streams = [], [], [torch.cuda.Stream(gpu) for _ in range(2)]
    for case, most in ((one, 1), (two, 90)):
        dev = [t.to(gpu) for t in case]
        ops.attn_paged(*dev, max_new=most)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.attn_paged(*dev, max_new=most))
        graphs.append((graph, dev))
    for _ in range(5):
        for o in outs:
            o.fill_(7.0)
        torch.cuda.synchronize()
        for s, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(4):
                    graph.replay()
        torch.cuda.synchronize()
        check_attn(outs[0], one)
        check_attn(outs[1], two)


def test_attention_on_two_streams_at_once(gpu):
    cases = [attn_inputs(4, [3000, 17, 900, 0], [n] * 4, 32, 8, 128, 16, torch.bfloat16, 72 + n) for n in (1, 24)]
    dev = [[t.to(gpu) for t in c] for c in cases]
    work = [ops.attn_paged_workspace(gpu) for _ in cases]
    want = [ops.attn_paged(*d, max_new=n, workspace=w) for d, n, w in zip(dev, (1, 24), work)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(gpu) for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.attn_paged(*dev[i], max_new=(1, 24)[i], workspace=work[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])
        check_attn(want[i], cases[i])


def test_decoder_in_half_precision(gpu):
    """The bf16 test's decoder with half-precision weights and caches (the activations of this model stay below 100), within
    8e-3 norm-wise: 16 half steps of 2^-11, where the bf16 bound of 2e-2 is 5 of 2^-8."""
    embed, blocks, final, head = model(gpu, 30)
    half = lambda t: t.half()
    blocks = [LlamaBlockWeights(*[half(getattr(b, f)) for f in ("input_norm", "qkv", "o", "post_norm", "gate_up", "down")])
              for b in blocks]
    m = (half(embed), blocks, half(final), half(head))
    text = torch.randint(0, V, (2, 45), generator=torch.Generator().manual_seed(8))
    want = [forward_fp32(m, t) for t in text]
    d = on(gpu, m)
    dec = PagedLlamaDecoder(d[0], d[1], d[2], d[3], NQ, NKV, D, max_len=64, slots=2, page_size=16)
    assert dec.k_cache[0].dtype == torch.float16 and len(dec.k_cache) == LAYERS
    at = [0, 0]
    for step in ([30, 1], [1, 40], [14, 4]):
        out = dec.append(torch.cat([text[r, at[r]:at[r] + n] for r, n in enumerate(step)]).to(gpu), step)
        t0 = 0
        for r, n in enumerate(step):
            assert rel(out[t0:t0 + n], want[r][at[r]:at[r] + n]) < 8e-3
            t0 += n
            at[r] += n
    tokens, n = dec.verify(text[:, 0].to(gpu), text[:, 1:4].to(gpu), torch.rand(2, 4, device=gpu), temperature=0.7, top_k=20, top_p=0.9)
    assert dec.lens.tolist() == [46 + n[0].item(), 46 + n[1].item()] and (tokens.gather(1, n[:, None]) >= 0).all()


def test_decoder_with_many_slots(gpu):
    """300 slots, every third one used, one token each after prompts of 1 to 9: rows against the fp32 pass."""
    mc = model(gpu, 31)
    m = on(gpu, mc)
    S, g = 300, torch.Generator().manual_seed(9)
    dec = PagedLlamaDecoder(m[0], m[1], m[2], m[3], NQ, NKV, D, max_len=16, slots=S, page_size=16, n_pages=100)
    lens = [1 + r % 9 if r % 3 == 0 else 0 for r in range(S)]
    text = torch.randint(0, V, (S, 10), generator=g)
    dec.append(torch.cat([text[r, :n] for r, n in enumerate(lens)]).to(gpu), lens)
    assert dec.granted.all() and dec.free_count.item() == 0
    live = [r for r in range(S) if lens[r]]
    out = dec.append(torch.stack([text[r, lens[r]] for r in live]).to(gpu), [1 if n else 0 for n in lens])
    for i in (0, 7, 50, 99):
        r = live[i]
        assert rel(out[i:i + 1], forward_fp32(mc, text[r, :lens[r] + 1])[-1:]) < 2e-2
    dec.append(text[1, :2].to(gpu), [0, 2] + [0] * (S - 2))               # no page left
    assert not dec.granted[1] and dec.granted.sum() == S - 1


def test_both_ways_to_the_current_stream_agree(gpu, monkeypatch):
    side = torch.cuda.Stream(gpu)
    assert ops._stream(gpu) == ops._public_stream(gpu.index)
    with torch.cuda.stream(side):
        assert ops._stream(gpu) == ops._public_stream(gpu.index) == side.cuda_stream
        monkeypatch.setattr(ops, "_raw_stream", ops._public_stream)       # as with a torch that lacks the short way
        x = torch.randn(3, 64, device=gpu)
        got = ops.rmsnorm(x, torch.ones(64, device=gpu), 1e-6)
    torch.cuda.synchronize()
    want = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    assert ((got - want).abs() <= 40 * 2.0 ** -24 * want.abs().amax()).all()  # 64 squares, a root, two products in fp32
