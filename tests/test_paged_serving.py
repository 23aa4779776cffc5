"""The paged decoder as a server uses it: requests that end at the longest length, idle slots, refused requests, drafts of
different lengths, calls that fail, models from the library."""
import pytest
import torch

from merak_amd import ops
from merak_amd.inference import PagedLlamaDecoder
from test_paged_decode import D, H, NKV, NQ, V, forward_fp32, model, on, rel


def gen(seed):
    return torch.Generator().manual_seed(52000 + seed)


def decoder(m, **kw):
    args = dict(max_len=128, slots=3, page_size=16)
    args.update(kw)
    return PagedLlamaDecoder(m[0], m[1], m[2], m[3], NQ, NKV, D, **args)


@pytest.mark.gpu
@pytest.mark.parametrize("max_len,page_size", [(100, 64), (33, 32), (17, 16), (64, 16)])
def test_a_request_ends_at_max_len(gpu, max_len, page_size):
    """The last page may have room behind max_len: a token there is refused like one that finds no page, whether it comes
    alone or with others, and the request goes on with what still fits.  bf16 activations: 2e-2 norm-wise, as for the
    other tests of this decoder."""
    m = model(gpu, 5)
    text = torch.randint(0, V, (2, max_len), generator=gen(max_len))
    want = [forward_fp32(m, t) for t in text]
    dec = decoder(on(gpu, m), max_len=max_len, page_size=page_size, slots=2)
    for c in dec.k_cache + dec.v_cache:
        c.fill_(50.0)                                    # what a released request may have left
    full = max_len - 2
    out = dec.append(torch.cat([text[0, :full], text[1, :3]]).to(gpu), [full, 3])
    assert dec.granted.all() and rel(out[:full], want[0][:full]) < 2e-2
    free = dec.free_count.item()
    out = dec.append(torch.cat([text[0, :3], text[1, 3:4]]).to(gpu), [3, 1])          # one token too many
    assert dec.granted.tolist() == [False, True] and dec.lens.tolist() == [full, 4]
    assert rel(out[3:], want[1][3:4]) < 2e-2
    out = dec.append(text[0, full:].to(gpu), [2, 0])
    assert dec.granted.all() and dec.lens.tolist() == [max_len, 4] and rel(out, want[0][full:]) < 2e-2
    dec.append(torch.cat([text[0, :1], text[1, 4:5]]).to(gpu), [1, 1])
    assert dec.granted.tolist() == [False, True] and dec.lens.tolist() == [max_len, 5]
    dec.append(text[0, :1].to(gpu), [1, 0])
    assert dec.granted.tolist() == [False, True] and dec.lens.tolist() == [max_len, 5]
    assert dec.held[0].item() == -(-max_len // page_size) and dec.free_count.item() <= free


@pytest.mark.gpu
def test_a_call_that_fails_leaves_the_state(gpu):
    """Tokens of another type, uniforms of another shape, more drafts than the verification takes, a temperature of zero:
    each raises, and the decoder goes on as if the call had not been made."""
    m = model(gpu, 6)
    text = torch.randint(0, V, (70,), generator=gen(1))
    want = forward_fp32(m, text)
    dec = decoder(on(gpu, m), slots=2)
    dec.append(text[:21].to(gpu), [21, 0])
    last, drafts, u = torch.zeros(2, dtype=torch.int64, device=gpu), torch.zeros(2, 3, dtype=torch.int64, device=gpu), \
        torch.full((2, 4), 0.5, device=gpu)
    many = torch.zeros(2, 65, dtype=torch.int64, device=gpu)
    state = lambda: [t.clone() for t in (dec.lens, dec.held, dec.free_count, dec.granted)]
    before = state()
    for call in (lambda: dec.append(text[21:30].int().to(gpu), [9, 0]),
                 lambda: dec.append(text[21:30], [9, 0]),                                   # not on the device
                 lambda: dec.step(text[21:30].int().to(gpu), [9, 0]),
                 lambda: dec.verify(last, drafts, u[:, :3]),
                 lambda: dec.verify(last, drafts, u.double()),
                 lambda: dec.verify(last, drafts, u, torch.zeros(2, 3, V - 1, device=gpu)),
                 lambda: dec.verify(last, drafts, u, temperature=0.0),
                 lambda: dec.verify(last, many, torch.full((2, 66), 0.5, device=gpu))):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()
        assert all(torch.equal(a, b) for a, b in zip(before, state()))
    out = dec.append(text[21:].to(gpu), [49, 0])
    assert dec.granted.all() and rel(out, want[21:]) < 2e-2


@pytest.mark.gpu
def test_refused_requests_give_no_tokens(gpu):
    """A pool too small for one request, then a request at max_len: step and verify say -1 and 0 for them, and the others
    get what a decoder without them gives."""
    m = on(gpu, model(gpu, 7))
    g = gen(3)
    text = torch.randint(0, V, (2, 40), generator=g).to(gpu)
    dec, alone = decoder(m, slots=2, n_pages=5), decoder(m, slots=1, n_pages=5)
    got = dec.step(torch.cat([text[0], text[1]]), [40, 40])               # three pages each, five in the pool
    assert dec.granted.tolist() == [True, False]
    want = alone.step(text[0], [40])
    assert got.tolist() == [want.item(), -1]
    drafts, u = torch.randint(0, V, (2, 12), generator=g).to(gpu), torch.rand(2, 13, generator=g).to(gpu)
    dec.append(text[1, :5], [0, 5])                                       # one page; the last one goes to the first request
    tokens, n = dec.verify(torch.stack([want[0], want[0]]), drafts, u, top_k=1)
    assert dec.granted.tolist() == [True, False] and n[1].item() == 0 and (tokens[1] == -1).all() and dec.lens[1].item() == 5
    t1, n1 = alone.verify(want, drafts[:1], u[:1], top_k=1)
    assert torch.equal(tokens[0], t1[0]) and n[0].item() == n1.item() and dec.lens[0].item() == alone.lens.item()
    full = decoder(m, slots=2, max_len=42)
    full.append(torch.cat([text[0], text[1, :3]]), [40, 3])
    tokens, n = full.verify(text[:, 0], drafts[:, :3], u[:, :4], top_k=1)
    assert full.granted.tolist() == [False, True] and (tokens[0] == -1).all() and n[0].item() == 0
    assert full.lens.tolist() == [40, 3 + 1 + n[1].item()]
    assert full.step(text[:, 0].repeat_interleave(torch.tensor([3, 1], device=gpu)), [3, 1])[0].item() == -1


@pytest.mark.gpu
def test_verify_leaves_idle_slots_alone(gpu):
    """A slot that was never used in front of the running one, and a released one behind it: they take no pages (the pool
    has none to spare), keep length 0 and start from nothing afterwards; the running request gets what it gets alone."""
    mc = model(gpu, 8)
    m = on(gpu, mc)
    g = gen(4)
    text = torch.randint(0, V, (3, 30), generator=g)
    dec, alone = decoder(m, slots=3, n_pages=5), decoder(m, slots=1, n_pages=3)
    dec.append(torch.cat([text[1], text[2]]).to(gpu), [0, 30, 30])
    dec.release([2])
    alone.append(text[1].to(gpu), [30])
    last = torch.tensor([3, 5, 7], device=gpu)
    for k in range(3):
        drafts, u = torch.randint(0, V, (3, 4), generator=g).to(gpu), torch.rand(3, 5, generator=g).to(gpu)
        tokens, n = dec.verify(last, drafts, u, top_k=1)
        t1, n1 = alone.verify(last[1:2], drafts[1:2], u[1:2], top_k=1)
        assert torch.equal(tokens[1], t1[0]) and n.tolist() == [0, n1.item(), 0]
        assert (tokens[0] == -1).all() and (tokens[2] == -1).all() and dec.granted.all()
        assert dec.lens.tolist() == [0, alone.lens.item(), 0] and dec.held.tolist() == [0, alone.held.item(), 0]
        last = torch.where(tokens >= 0, tokens, 0).gather(1, n[:, None]).squeeze(1)
    out = dec.append(text[2, :20].to(gpu), [0, 0, 20])
    assert dec.granted.all() and rel(out, forward_fp32(mc, text[2])[:20]) < 2e-2


@pytest.mark.gpu
def test_verify_with_drafts_of_different_lengths(gpu):
    """No slots, some drafts, none, all of them: each request gets what it gets alone with that many; slots left out stay,
    an empty slot that is named takes part, and a request that ends at max_len finishes with the drafts that fit."""
    m = on(gpu, model(gpu, 9))
    g = gen(5)
    K, text = 4, torch.randint(0, V, (4, 25), generator=g).to(gpu)
    lens = [25, 11, 0, 20]
    dec = decoder(m, slots=4, max_len=27, n_pages=8)
    dec.append(torch.cat([text[r, :n] for r, n in enumerate(lens)]), lens)
    drafts, u = torch.randint(0, V, (4, K), generator=g).to(gpu), torch.rand(4, K + 1, generator=g).to(gpu)
    guess = torch.softmax(torch.randn(4, K, V, generator=g) * 3, -1).to(gpu)
    last = text[:, 3]
    tokens, n = dec.verify(last, drafts, u, draft_lens=[-1] * 4)
    assert (tokens == -1).all() and not n.any() and dec.lens.tolist() == lens and dec.granted.all()
    tokens, n = dec.verify(last, drafts, u, draft_lens=[K, -1, -1, -1])   # five tokens where two fit
    assert dec.granted.tolist() == [False, True, True, True] and (tokens == -1).all() and dec.lens.tolist() == lens
    for probs in (None, guess):
        want = [1, K, 0, -1]
        before = dec.lens.tolist()
        tokens, n = dec.verify(last, drafts, u, probs, top_k=1, draft_lens=want)
        after = dec.lens.tolist()
        for r in range(4):
            if want[r] < 0:
                assert (tokens[r] == -1).all() and n[r].item() == 0 and after[r] == before[r]
                continue
            one = decoder(m, slots=1, max_len=27)
            if lens[r]:
                one.append(text[r, :lens[r]], [lens[r]])
            k = want[r]
            t1, n1 = one.verify(last[r:r + 1], drafts[r:r + 1, :k], torch.cat([u[r:r + 1, :k], u[r:r + 1, K:]], 1),
                                None if probs is None else probs[r:r + 1, :k], top_k=1, draft_lens=[k])
            assert dec.granted[r] and n[r].item() == n1.item() <= k and after[r] == before[r] + 1 + n1.item()
            assert tokens[r].tolist() == t1[0].tolist() + [-1] * (K - k)
        dec.release(range(4))
        dec.append(torch.cat([text[r, :n] for r, n in enumerate(lens)]), lens)
    for bad in ([K + 1, 0, 0, 0], [0, 0, 0], [-2, 0, 0, 0]):
        with pytest.raises(ValueError, match="draft_lens"):
            dec.verify(last, drafts, u, draft_lens=bad)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", [0, 1])
def test_speculative_steps_against_the_targets_own_logits(gpu, seed):
    """top_k = 1 makes the target certain.  Every accepted draft and every drawn token is the argmax of the target's logits
    at its position (from a decoder that got the text in one piece), every rejected draft is not; a request whose drafts
    are those argmaxes has all of them accepted.  Positions whose two largest logits lie within the 2e-2 of the other
    tests (norm-wise: of the root mean square of a row, on either side) are not judged."""
    mc = model(gpu, 20 + seed)
    m = on(gpu, mc)
    g = gen(seed + 6)
    prompt = torch.randint(0, V, (2, 17), generator=g)
    dec = decoder(m, slots=2)
    first = dec.step(prompt.reshape(-1).to(gpu), [17, 17]).cpu()
    text = [prompt[r].tolist() + [int(first[r])] for r in range(2)]        # the last token is not in the cache yet
    K, judged, all_kept = 4, 0, 0

    def logits(seq):
        return torch.nn.functional.linear(forward_fp32(mc, torch.tensor(seq)), mc[3].float())

    def sure(row):
        top = row.topk(2).values
        return (top[0] - top[1]).item() > 2 * 2e-2 * row.square().mean().sqrt().item()

    for _ in range(6):
        greedy = list(text[0])                                            # the first request's drafts: its own argmaxes
        clear = True
        for _ in range(K):
            row = logits(greedy)[-1]
            clear &= sure(row)
            greedy.append(int(row.argmax()))
        clear &= sure(logits(greedy)[-1])
        drafts = torch.stack([torch.tensor(greedy[-K:]), torch.randint(0, V, (K,), generator=g)])
        if judged % 2:                                                    # the second request: one right draft, then noise
            drafts[1, 0] = int(logits(text[1])[-1].argmax())
        last = torch.tensor([t[-1] for t in text])
        tokens, n = dec.verify(last.to(gpu), drafts.to(gpu), torch.rand(2, K + 1, generator=g).to(gpu), top_k=1)
        tokens, n = tokens.cpu(), n.tolist()
        if clear:
            assert n[0] == K
            all_kept += 1
        for r in range(2):
            rows = logits(text[r] + drafts[r].tolist())[len(text[r]) - 1:]   # of the last token, then behind each draft
            for i in range(n[r]):
                assert int(tokens[r, i]) == int(drafts[r, i])
                assert not sure(rows[i]) or int(drafts[r, i]) == int(rows[i].argmax())
            at = rows[n[r]]
            if sure(at):
                judged += 1
                assert int(tokens[r, n[r]]) == int(at.argmax())
                assert n[r] == K or int(drafts[r, n[r]]) != int(at.argmax())
            assert (tokens[r, n[r] + 1:] == -1).all()
            text[r] += tokens[r, :n[r] + 1].tolist()
            assert dec.lens[r].item() == len(text[r]) - 1
    assert judged >= 8 and all_kept >= 3, (judged, all_kept)
