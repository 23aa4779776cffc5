"""Operators of serving over a paged key/value cache, and the query/key norm with rotary embedding that training shares
with it: what they compute in plain torch, the calls a user makes of them, and the sizes they are measured at.

Five kinds of case, one operator each:

``plan``    pages handed to requests, cumulative token counts, positions and cache slots of a step, on the device
``rotary``  RMSNorm of each query and key head and rotary embedding, forward and backward (training)
``append``  the same for serving: rotated queries out, keys and values into the pages of a cache
``attn``    causal attention of a chunk of new tokens per request over the pages of its cache
``verify``  drafted tokens accepted or rejected against the target's probabilities, and the token drawn after them

``own`` false: elementary torch operations in 32 bits (64 for cumulative sums that decide a token), rounded once.
``own`` true: the calls into ``merak_amd``.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_EPS = 1e-5


def _ops():
    from merak_amd import ops
    return ops


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one decode step of a full batch: every request adds one token, few of them a page
        {"name": "plan decode 256", "op": "plan", "requests": 256, "len_lo": 1, "len_hi": 16000, "new_lo": 1, "new_hi": 1, "page": 16},
        # a step that mixes fresh prompts and running requests
        {"name": "plan prompts 512", "op": "plan", "requests": 512, "len_lo": 0, "len_hi": 4000, "new_lo": 1, "new_hi": 611, "page": 64},
        # one training micro batch of an 8B-shaped layer: 32 query and 8 key heads of 128
        {"name": "rotary train 8192", "op": "rotary", "dtype": "bf16", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "norm": True},
        # a small fp32 model with as many key as query heads of 64, odd token count
        {"name": "rotary train f32 1001", "op": "rotary", "dtype": "f32", "tokens": 1001, "heads": 12, "kv_heads": 12, "dim": 64, "norm": True},
        # one token of each of 32 requests, on its way into the cache: the smallest launch
        {"name": "append decode 32", "op": "append", "dtype": "bf16", "tokens": 32, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "norm": True},
        # a prompt of one tensor-parallel rank of eight of a 70B-shaped model, half precision, odd length
        {"name": "append prompt 8191", "op": "append", "dtype": "f16", "tokens": 8191, "heads": 8, "kv_heads": 1, "dim": 128, "page": 64, "norm": False},
        # decode: one new token per request, lengths from short to long
        {"name": "attn decode 64", "op": "attn", "dtype": "bf16", "requests": 64, "heads": 32, "kv_heads": 8, "dim": 128, "len_lo": 200, "len_hi": 8192, "new_lo": 1, "new_hi": 1, "page": 16},
        # one request far into a long context
        {"name": "attn long 1", "op": "attn", "dtype": "bf16", "requests": 1, "heads": 32, "kv_heads": 8, "dim": 128, "len_lo": 130001, "len_hi": 130001, "new_lo": 1, "new_hi": 1, "page": 64},
        # five tokens per request: four drafts and the last accepted token, to be verified together
        {"name": "attn drafts 32", "op": "attn", "dtype": "f16", "requests": 32, "heads": 32, "kv_heads": 8, "dim": 128, "len_lo": 500, "len_hi": 6000, "new_lo": 5, "new_hi": 5, "page": 32},
        # prompts in chunks behind what is cached already
        {"name": "attn prompts 4", "op": "attn", "dtype": "bf16", "requests": 4, "heads": 32, "kv_heads": 8, "dim": 128, "len_lo": 1, "len_hi": 5000, "new_lo": 1900, "new_hi": 4100, "page": 16},
        # a few requests of an interactive server, drafts from a smaller model with its own probabilities
        {"name": "verify 8 x 4", "op": "verify", "dtype": "f32", "requests": 8, "drafts": 4, "vocab": 128256, "draft_probs": True},
        # a full batch with drafts looked up in the prompt (no probabilities of their own), odd vocabulary
        {"name": "verify 128 x 7", "op": "verify", "dtype": "f32", "requests": 128, "drafts": 7, "vocab": 50257, "draft_probs": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "rotary", "append", "attn", "attn", "verify"])
    heads, kv = rng.choice([(32, 8), (8, 1), (12, 12), (64, 8), (16, 2), (7, 7), (28, 4)])
    dim = rng.choice([64, 128])
    page = rng.choice([16, 32, 64, 128])
    half = rng.choice(["bf16", "f16"])
    if op == "plan":
        new_lo = rng.choice([0, 1, 1])
        return {"op": op, "requests": _log(rng, 1, 700), "len_lo": 0, "len_hi": _log(rng, 10, 16000), "new_lo": new_lo,
                "new_hi": 1 if rng.random() < 0.4 else _log(rng, 2, 400), "page": page}
    if op == "rotary":
        return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]), "tokens": _log(rng, 1, 4000), "heads": heads, "kv_heads": kv,
                "dim": dim, "norm": rng.random() < 0.7}
    if op == "append":
        return {"op": op, "dtype": half, "tokens": _log(rng, 1, 8000), "heads": heads, "kv_heads": kv, "dim": dim, "page": page,
                "norm": rng.random() < 0.5}
    if op == "attn":
        kind = rng.choice(["decode", "drafts", "prompts", "mixed"])
        if kind == "decode":
            r, hi, new = _log(rng, 1, 96), _log(rng, 2, 8000), (1, 1)
        elif kind == "drafts":
            r, hi, new = _log(rng, 1, 32), _log(rng, 30, 8000), (2, rng.randint(3, 17))
        elif kind == "prompts":
            r, hi, new = rng.randint(1, 4), _log(rng, 30, 5000), (rng.randint(20, 200), _log(rng, 300, 2500))
        else:
            r, hi, new = _log(rng, 2, 24), _log(rng, 30, 4000), (0, _log(rng, 20, 700))
        return {"op": op, "dtype": half, "requests": r, "heads": heads, "kv_heads": kv, "dim": dim, "len_lo": rng.randint(0, min(hi, 60)),
                "len_hi": hi, "new_lo": new[0], "new_hi": new[1], "page": page}
    return {"op": op, "dtype": rng.choice(["f32", "f32", "bf16"]), "requests": _log(rng, 1, 96), "drafts": rng.randint(1, 9),
            "vocab": _log(rng, 200, 60000), "draft_probs": rng.random() < 0.6}


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spaced over their logarithm: the same total work for every seed."""
    if n == 1:
        return [hi]
    return [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** (i / (n - 1)))) - 1 for i in range(n)]


def _ceil(a, b):
    return -(-a // b)


def _shuffled(values, gen):
    return [values[i] for i in torch.randperm(len(values), generator=gen).tolist()]


def _lens(case, gen):
    """Cached and new tokens of each request, in an order made from the seed."""
    r = case["requests"]
    return (_shuffled(_spread(case["len_lo"], case["len_hi"], r), gen), _shuffled(_spread(case["new_lo"], case["new_hi"], r), gen))


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    cpu = torch.Generator().manual_seed(seed)
    gpu = torch.Generator(device=dev).manual_seed(seed)

    def normal(shape, dtype, scale=1.0):
        return torch.randn(shape, generator=gpu, device=dev).mul_(scale).to(dtype)

    st = {"case": case}
    op = case["op"]
    if op == "plan":
        page, n = case["page"], case["requests"]
        lens, new = _lens(case, cpu)
        held = [_ceil(a, page) for a in lens]
        cols = _ceil(case["len_hi"] + case["new_hi"], page) + 3
        need = sum(max(0, _ceil(a + b, page) - h) for a, b, h in zip(lens, new, held))
        used, spare = sum(held), need + 5
        ids = torch.randperm(used + spare, generator=cpu).to(torch.int32)
        table = torch.full((n, cols), -1, dtype=torch.int32)
        at = 0
        for r, h in enumerate(held):
            table[r, :h] = ids[at:at + h]
            at += h
        free = torch.full((used + spare,), -1, dtype=torch.int32)
        free[:spare] = ids[used:]
        i64 = lambda v: torch.tensor(v, dtype=torch.int64, device=dev)
        st.update(lens=i64(lens), new=i64(new), held=torch.tensor(held, dtype=torch.int32, device=dev), table=table.to(dev),
                  free=free.to(dev), count=torch.tensor([spare], dtype=torch.int32, device=dev), tokens=sum(new),
                  most=max(new) // page + 1)
        return st
    if op in ("rotary", "append"):
        t, hq, hk, d, dt = case["tokens"], case["heads"], case["kv_heads"], case["dim"], _DT[case["dtype"]]
        longest = t + 700
        freq = 500000.0 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
        ang = torch.arange(longest, device=dev, dtype=torch.float64)[:, None] * freq
        ang = torch.cat([ang, ang], 1)
        st.update(qkv=normal((t, (hq + 2 * hk) * d), dt), cos=ang.cos().float(), sin=ang.sin().float(),
                  positions=(torch.arange(t, device=dev) + int(torch.randint(0, 700, (1,), generator=cpu))))
        if case["norm"]:
            st.update(qw=(normal((d,), torch.float32, 0.1) + 1.0).to(dt), kw=(normal((d,), torch.float32, 0.1) + 1.0).to(dt))
        else:
            st.update(qw=None, kw=None)
        if op == "rotary":
            st.update(dq=normal((t, hq, d), dt), dk=normal((t, hk, d), dt), dv=normal((t, hk, d), dt))
            return st
        page = case["page"]
        pages = _ceil(t, page) + 4
        at = torch.randperm(pages, generator=cpu)[:_ceil(t, page)].to(dev)
        j = torch.arange(t, device=dev)
        st.update(slots=at[j // page] * page + j % page, k_cache=normal((pages, hk, page, d), dt), v_cache=normal((pages, hk, page, d), dt))
        return st
    if op == "attn":
        hq, hk, d, dt, page = case["heads"], case["kv_heads"], case["dim"], _DT[case["dtype"]], case["page"]
        lens, new = _lens(case, cpu)
        kv = [a + b for a, b in zip(lens, new)]
        rows = [_ceil(a, page) for a in kv]
        pages = sum(rows) + 3
        ids = torch.randperm(pages, generator=cpu).to(torch.int32)
        table = torch.full((len(kv), max(rows) + 1), -1, dtype=torch.int32)
        at = 0
        for r, h in enumerate(rows):
            table[r, :h] = ids[at:at + h]
            at += h
        cu = [0]
        for b in new:
            cu.append(cu[-1] + b)
        st.update(q=normal((cu[-1], hq, d), dt), k_cache=normal((pages, hk, page, d), dt), v_cache=normal((pages, hk, page, d), dt),
                  table=table.to(dev), cu=torch.tensor(cu, dtype=torch.int64, device=dev),
                  kv=torch.tensor(kv, dtype=torch.int64, device=dev), host_new=new, host_kv=kv, max_new=max(new), bound=max(kv))
        if own:
            st["workspace"] = _ops().attn_paged_workspace(dev)
        return st
    r, k, v, dt = case["requests"], case["drafts"], case["vocab"], _DT[case["dtype"]]
    logits = torch.randn((r, k + 1, v), generator=gpu, device=dev).mul_(3.0)
    target = torch.softmax(logits, -1).to(dt)
    guess = torch.softmax(logits[:, :k] + torch.randn((r, k, v), generator=gpu, device=dev).mul_(0.4), -1).to(dt)
    u = torch.rand((r, k, 1), generator=gpu, device=dev, dtype=torch.float64)
    cum = guess.double().cumsum(-1)
    if case["draft_probs"]:      # drafts drawn from the draft model's own probabilities
        drafts = torch.searchsorted(cum, u * cum[..., -1:]).squeeze(-1).clamp_max(v - 1)
    else:                        # drafts found elsewhere: mostly the likeliest token
        drafts = torch.where(u.squeeze(-1) < 0.8, target[:, :k].float().argmax(-1), (u.squeeze(-1) * v).long())
    st.update(drafts=drafts, target=target, guess=guess if case["draft_probs"] else None,
              uniforms=torch.rand((r, k + 1), generator=gpu, device=dev))
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    ops = _ops()
    op = s["case"]["op"]
    if op == "plan":
        p = ops.paged_plan(s["lens"], s["new"], s["held"], s["table"], s["free"], s["count"], s["case"]["page"], s["tokens"])
        return [p.slots, p.positions, p.cu, p.kv_lens, p.granted, p.held, p.free_count, s["table"]]
    if op == "rotary":
        q, k = ops.qk_norm_rope(s["qkv"], s["cos"], s["sin"], s["positions"], s["case"]["heads"], s["qw"], s["kw"], _EPS)
        dqkv, dqw, dkw = ops.qk_norm_rope_bwd(s["dq"], s["dk"], s["dv"], s["qkv"], s["cos"], s["sin"], s["positions"], s["qw"], s["kw"], _EPS)
        return [q, k, dqkv] + ([dqw, dkw] if s["case"]["norm"] else [])
    if op == "append":
        q = ops.qk_norm_rope_append(s["qkv"], s["cos"], s["sin"], s["positions"], s["slots"], s["k_cache"], s["v_cache"],
                                    s["case"]["heads"], s["qw"], s["kw"], _EPS)
        return [q, s["k_cache"], s["v_cache"]]
    if op == "attn":
        return ops.attn_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["kv"], max_new=s["max_new"],
                              len_bound=s["bound"], workspace=s.get("workspace"))
    tokens, accepted = ops.verify_draft(s["drafts"], s["target"], s["guess"], s["uniforms"])
    return [tokens, accepted]


def _run_plain(s):
    return {"plan": _plain_plan, "rotary": _plain_rotary, "append": _plain_append, "attn": _plain_attn, "verify": _plain_verify}[
        s["case"]["op"]](s)


def _plain_plan(s):
    page, cap = s["case"]["page"], s["tokens"]
    lens, table, dev = s["lens"], s["table"], s["lens"].device
    cols = table.shape[1]
    new = s["new"].clamp(0, cap + 1)
    held = s["held"].long()
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    fits = (lens >= 0) & (held >= 0) & (held <= cols) & (lens + new <= cols * page) & (cu[1:] <= cap)
    need = torch.where(fits, ((lens + new + page - 1) // page - held).clamp_min(0), 0)
    upto = need.cumsum(0)
    count = s["count"].long().clamp(0, s["free"].shape[0])
    granted = fits & ((need == 0) | (upto <= count))
    take = torch.where(granted, need, 0)
    # the i-th page handed out is the i-th from the top of the free list
    j = torch.arange(s["most"], device=dev)
    rank = (upto - need)[:, None] + j
    gives = j < take[:, None]
    ids = s["free"][(count - 1 - rank).clamp_min(0)]
    at = (held[:, None] + j).clamp_max(cols - 1)
    table.scatter_(1, at, torch.where(gives, ids, table.gather(1, at)))
    t = torch.arange(cap, device=dev)
    r = torch.searchsorted(cu[1:], t, right=True)
    inside = r < lens.shape[0]
    r = r.clamp_max(lens.shape[0] - 1)
    inside &= granted[r]
    pos = lens[r] + t - cu[r]
    ok_pos = torch.where(inside, pos, 0)
    ids = table[r, ok_pos // page].long()
    slots = torch.where(inside, ids * page + ok_pos % page, -1)
    return [slots, torch.where(inside, pos, -1), cu, torch.where(granted, lens + new, 0), granted, (held + take).int(),
            (count - take.sum()).int(), table]


def _turn(x, cos, sin):
    h = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., h:], x[..., :h]], -1) * sin


def _plain_heads(s):
    c = s["case"]
    x = s["qkv"].float().view(c["tokens"], c["heads"] + 2 * c["kv_heads"], c["dim"])
    return x[:, :c["heads"]], x[:, c["heads"]:c["heads"] + c["kv_heads"]]


def _plain_norm_rope(x, w, cos, sin):
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w.float()
    return _turn(x, cos, sin)


def _plain_rotary(s):
    c, dt = s["case"], s["qkv"].dtype
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    half = c["dim"] // 2
    outs, grads, dws = [], [], []
    for x, w, dy in zip(_plain_heads(s), (s["qw"], s["kw"]), (s["dq"], s["dk"])):
        outs.append(_plain_norm_rope(x, w, cos, sin).to(dt))
        dy = dy.float()
        a = dy * sin
        dz = dy * cos + torch.cat([a[..., half:], -a[..., :half]], -1)
        if w is None:
            grads.append(dz)
            continue
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        n = x * r
        dws.append((dz * n).sum((0, 1)).to(dt))
        dn = dz * w.float()
        grads.append(r * (dn - n * (dn * n).mean(-1, keepdim=True)))
    dqkv = torch.cat(grads + [s["dv"].float()], 1).to(dt).view(c["tokens"], -1)
    return outs + [dqkv] + dws


def _plain_append(s):
    c, dt, page = s["case"], s["qkv"].dtype, s["case"]["page"]
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    q, k = (_plain_norm_rope(x, w, cos, sin).to(dt) for x, w in zip(_plain_heads(s), (s["qw"], s["kw"])))
    p, o = s["slots"] // page, s["slots"] % page
    s["k_cache"][p, :, o] = k
    s["v_cache"][p, :, o] = s["qkv"].view(c["tokens"], -1, c["dim"])[:, c["heads"] + c["kv_heads"]:]
    return [q, s["k_cache"], s["v_cache"]]


def _plain_attn(s):
    c = s["case"]
    hq, hk, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    g = hq // hk
    out = torch.zeros_like(s["q"])
    t0 = 0
    for r, (n, kv) in enumerate(zip(s["host_new"], s["host_kv"])):
        if n == 0:
            continue
        ids = s["table"][r, :_ceil(kv, page)].long()
        k, v = (x[ids].transpose(0, 1).reshape(hk, -1, d)[:, :kv].float() for x in (s["k_cache"], s["v_cache"]))
        i = torch.arange(n, device=k.device)
        mask = torch.arange(kv, device=k.device)[None, :] > (kv - n + i)[:, None]
        for h in range(hk):
            q = s["q"][t0:t0 + n, h * g:(h + 1) * g].float().transpose(0, 1).reshape(g * n, d)
            x = (q @ k[h].t().contiguous()) * d ** -0.5
            x = x.view(g, n, kv).masked_fill(mask, -math.inf)
            e = torch.exp(x - x.amax(-1, keepdim=True))
            o = (e / e.sum(-1, keepdim=True)).view(g * n, kv) @ v[h]
            out[t0:t0 + n, h * g:(h + 1) * g] = o.view(g, n, d).transpose(0, 1).to(out.dtype)
        t0 += n
    return out


def _plain_verify(s):
    k = s["case"]["drafts"]
    target, guess, drafts, u = s["target"], s["guess"], s["drafts"], s["uniforms"].double()
    p = target[:, :k].gather(2, drafts[..., None]).squeeze(-1).double()
    q = torch.ones_like(p) if guess is None else guess.gather(2, drafts[..., None]).squeeze(-1).double()
    ok = u[:, :k] * q < p
    n = ok.long().cumprod(1).sum(1)
    rows = torch.arange(n.shape[0], device=n.device)
    w = target[rows, n].double()
    at = n.clamp_max(k - 1)
    minus = torch.zeros_like(w).scatter_(1, drafts[rows, at][:, None], math.inf) if guess is None else guess[rows, at].double()
    left = (w - minus).clamp_min(0)
    left = torch.where((left.sum(1) > 0)[:, None], left, w)
    w = torch.where((n < k)[:, None], left, w)
    cum = w.cumsum(1)
    token = (cum <= u[:, k:] * cum[:, -1:]).sum(1)
    tokens = torch.where(torch.arange(k + 1, device=n.device) < n[:, None], torch.cat([drafts, drafts[:, :1]], 1), -1)
    tokens[rows, n] = token
    return [tokens, n]


# ------------------------------------------------------------------------------------------------ least work
def work(case):
    op = case["op"]
    if op == "plan":
        r, t = case["requests"], sum(_spread(case["new_lo"], case["new_hi"], case["requests"]))
        # lens, new, held in; cu, kv_lens, granted, held out; per token its page, slot and position
        return {"bytes": r * (8 + 8 + 4 + 8 + 8 + 1 + 4) + t * (8 + 8) + 4 * _ceil(t, case["page"]) * 2, "flops": 0}
    if op in ("rotary", "append"):
        t, d, e = case["tokens"], case["dim"], 4 if case["dtype"] == "f32" else 2
        hq, hk = case["heads"], case["kv_heads"]
        table = t * 2 * d * 4
        if op == "append":
            return {"bytes": 2 * t * (hq + 2 * hk) * d * e + table + 16 * t, "flops": t * (hq + hk) * d * 8}
        fwd = 2 * t * (hq + hk) * d * e
        bwd = t * (hq + hk) * d * e + 2 * t * (hq + 2 * hk) * d * e
        # one pass through the operator is a forward and a backward: the backward cannot reuse what the forward read
        return {"bytes": fwd + bwd + 2 * (table + 8 * t), "flops": t * (hq + hk) * d * 28}
    if op == "attn":
        lens = _spread(case["len_lo"], case["len_hi"], case["requests"])
        new = _spread(case["new_lo"], case["new_hi"], case["requests"])
        hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
        # the order of the seed pairs lengths and new tokens at random: the mean over all pairs
        mean = sum(lens) / len(lens)
        pairs = sum(b * (mean + (b + 1) / 2) for b in new)
        return {"bytes": int(sum(lens) + sum(new)) * hk * d * 2 * 2 + 2 * sum(new) * hq * d * 2, "flops": int(pairs * hq * d * 4)}
    r, k, v, e = case["requests"], case["drafts"], case["vocab"], 4 if case["dtype"] == "f32" else 2
    # one row of the target per request, one of the draft where a draft was rejected (about two requests in three)
    return {"bytes": int(r * v * e * (5 / 3 if case["draft_probs"] else 1)) + r * (k + 1) * 24, "flops": r * v * 4}


# ------------------------------------------------------------------------------------------------ by definition
def exact(case, seed):
    """What run() returns, from the definitions: whole numbers by loops on the host, the rest in 64 bits."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        page, cap = case["page"], s["tokens"]
        lens, new, held, table, free = (s[n].tolist() for n in ("lens", "new", "held", "table", "free"))
        stack = free[:s["count"].item()]
        slots, positions, cu, kv, granted, short = [-1] * cap, [-1] * cap, [0], [], [], False
        for r in range(len(lens)):
            cu.append(cu[-1] + new[r])
            need = max(0, _ceil(lens[r] + new[r], page) - held[r])
            good = lens[r] + new[r] <= len(table[r]) * page and cu[-1] <= cap
            if good and need and (short or need > len(stack)):
                short, good = True, False
            granted.append(good)
            kv.append(lens[r] + new[r] if good else 0)
            if not good:
                continue
            for _ in range(need):
                table[r][held[r]] = stack.pop()
                held[r] += 1
            for i in range(new[r]):
                pos = lens[r] + i
                positions[cu[r] + i] = pos
                slots[cu[r] + i] = table[r][pos // page] * page + pos % page
        dev = s["lens"].device
        mk = lambda v, t=torch.int64: torch.tensor(v, dtype=t, device=dev)
        return [mk(slots), mk(positions), mk(cu), mk(kv), mk(granted, torch.bool), mk(held, torch.int32), mk([len(stack)], torch.int32),
                mk(table, torch.int32)]
    if op in ("rotary", "append"):
        t, hq, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        x = s["qkv"].double().view(t, hq + 2 * hk, d)
        # as complex numbers: (x1 + i x2) e^{i angle}, both halves of the tables being equal
        cis = torch.complex(s["cos"][s["positions"], :d // 2].double(), s["sin"][s["positions"], :d // 2].double())[:, None]
        both = lambda z: torch.cat([z.real, z.imag], -1)
        pair = lambda a: torch.complex(a[..., :d // 2].contiguous(), a[..., d // 2:].contiguous())
        outs, grads, dws = [], [], []
        for a, w, dy in ((x[:, :hq], s["qw"], s.get("dq")), (x[:, hq:hq + hk], s["kw"], s.get("dk"))):
            scale = 1.0 if w is None else (a.square().sum(-1, keepdim=True) / d + _EPS).pow(-0.5)
            unit = a * scale
            z = unit if w is None else unit * w.double()
            outs.append(both(pair(z) * cis))
            if dy is None:
                continue
            dz = both(pair(dy.double()) * cis.conj())
            if w is not None:
                dws.append(torch.einsum("thd,thd->d", dz, unit))
                dz = dz * w.double()
                dz = scale * dz - scale * unit * torch.einsum("thd,thd->th", dz, unit)[..., None] / d
            grads.append(dz)
        if op == "rotary":
            return outs + [torch.cat(grads + [s["dv"].double()], 1).view(t, -1)] + dws
        page, done = case["page"], []
        for cache, rows in ((s["k_cache"], outs[1]), (s["v_cache"], x[:, hq + hk:])):
            flat = cache.double().transpose(1, 2).reshape(-1, hk, d).clone()       # a row for each slot
            flat[s["slots"]] = rows
            done.append(flat.view(-1, page, hk, d).transpose(1, 2).contiguous())
        return [outs[0]] + done
    if op == "attn":
        hq, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
        g, out, t0 = hq // hk, torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device), 0
        for r, (n, kv) in enumerate(zip(s["host_new"], s["host_kv"])):
            j = torch.arange(kv, device=out.device)
            where = s["table"][r].long()[j // page]
            for h in range(hk):
                k, v = s["k_cache"][where, h, j % page].double(), s["v_cache"][where, h, j % page].double()
                for a in range(0, n, 512):       # rows at a time: a matrix of scores stays small
                    b = min(n, a + 512)
                    seen = kv - n + b            # what the last of these rows sees
                    for e in range(h * g, (h + 1) * g):
                        x = torch.mm(s["q"][t0 + a:t0 + b, e].double(), k[:seen].t().contiguous()) / math.sqrt(d)
                        x += torch.full_like(x, -math.inf).triu_(kv - n + a + 1)
                        out[t0 + a:t0 + b, e] = torch.mm((x - x.logsumexp(1, keepdim=True)).exp(), v[:seen])
            t0 += n
        return out
    import numpy as np
    k, v = case["drafts"], case["vocab"]
    drafts, u = s["drafts"].cpu().numpy(), s["uniforms"].double().cpu().numpy()
    tokens, counts = [], []
    for r in range(case["requests"]):
        line, n = [], 0
        while n < k:
            x = int(drafts[r, n])
            p = float(s["target"][r, n, x])
            q = 1.0 if s["guess"] is None else float(s["guess"][r, n, x])
            if not u[r, n] * q < p:
                break
            line.append(x)
            n += 1
        w = s["target"][r, n].double().cpu().numpy()
        if n < k:
            if s["guess"] is None:
                rest = w.copy()
                rest[int(drafts[r, n])] = 0.0
            else:
                rest = np.maximum(w - s["guess"][r, n].double().cpu().numpy(), 0.0)
            w = rest if rest.sum() > 0 else w
        total = np.cumsum(w)
        line.append(int(np.searchsorted(total, u[r, k] * total[-1], side="right")))
        tokens.append(line + [-1] * (k + 1 - len(line)))
        counts.append(n)
    dev = s["drafts"].device
    return [torch.tensor(tokens, device=dev), torch.tensor(counts, device=dev)]
