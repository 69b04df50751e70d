"""Cases for measuring the key/value cache operators: the cache in 16 or 8 bits, and attention of new tokens over it.

With `own` false `run` computes the plain form in elementary torch operations; with `own` true it calls the package.
The 8-bit formats hold a head row in blocks of 32 elements that share a power-of-two scale 2^e: e is the smallest integer
(-100 at least) with max |x| <= top 2^e, top = 448 (e4m3) or 127 (int8), and an element is held as x 2^-e rounded to nearest even.
"""
import math

import torch

own = False

TOP = {"e4m3": 448.0, "int8": 127.0}
PAGE = 64
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------- cases
def _attend(name, fmt, heads, kv, dim, seqs, new, ctx, window=0):
    """`seqs` sequences; sequence lengths are spread between ctx / 2 and ctx, new tokens between new / 2 and new (ragged > 1)."""
    c = dict(kind="attend", fmt=fmt, heads=heads, kv=kv, dim=dim, seqs=seqs, new=new, ctx=ctx, window=window, io="bf16")
    return dict(c, name=name) if name else c


def _cache(name, fmt, kv, dim, seqs, new, ctx, io):
    c = dict(kind="cache", fmt=fmt, heads=kv, kv=kv, dim=dim, seqs=seqs, new=new, ctx=ctx, window=0, io=io)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one utterance, one new token behind a short prompt: the smallest call, where only latency counts
        _attend("token_alone", "bf16", 16, 8, 128, 1, 1, 113),
        # the talker's decode step at the benchmark's batch and length
        _attend("tokens_talker", "e4m3", 16, 8, 128, 64, 1, 500),
        # few sequences with long contexts: the walk over the keys has to be split
        _attend("tokens_long_int8", "int8", 32, 8, 128, 12, 1, 30011),
        # the same in 16 bits, one query head group of eight on a single key head
        _attend("tokens_long_bf16", "bf16", 8, 1, 128, 7, 1, 20011),
        # five drafted tokens per sequence scored at once
        _attend("drafts_int8", "int8", 16, 8, 128, 32, 5, 2047),
        # a long prompt from nothing
        _attend("prompt_bf16", "bf16", 16, 8, 128, 2, 4096, 4096),
        # the next part of long prompts, ragged and odd, behind what the cache holds already
        _attend("chunk_e4m3", "e4m3", 32, 8, 128, 3, 509, 15013),
        # sliding window of the codec's transformer over whole utterances
        _attend("window_bf16", "bf16", 16, 16, 64, 24, 375, 375, window=72),
        # one frame's keys and values joined to 64 utterances
        _cache("append_int8", "int8", 8, 128, 64, 1, 250, "bf16"),
        # prompts that arrive in f32
        _cache("prompts_e4m3", "e4m3", 8, 128, 5, 2011, 2011, "f32"),
        # long sequences at once
        _cache("sequences_int8", "int8", 8, 128, 16, 8192, 8192, "bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    most_bytes, most_flops = 8.0e8, 3.0e11
    while True:
        dim = rng.choice([64, 128])
        if rng.random() < 0.7:
            kv = rng.choice([1, 2, 4, 8, 16])
            heads = kv * rng.choice([1, 2, 3, 4, 5, 8])
            fmt = rng.choice(["bf16", "e4m3", "int8"])
            new = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 4096)])
            ctx = max(new, _log(rng, 1, 32000))
            seqs = _log(rng, 1, 96)
            window = rng.choice([0, 0, 0, _log(rng, 1, 1024)])
            case = _attend(None, fmt, heads, kv, dim, seqs, new, ctx, window)
        else:
            new = rng.choice([1, _log(rng, 2, 8192)])
            case = _cache(None, rng.choice(["bf16", "e4m3", "int8"]), rng.choice([1, 2, 4, 8, 16]), dim, _log(rng, 1, 96), new,
                          max(new, _log(rng, 1, 8192)), rng.choice(["bf16", "f32"]))
        w = work(case)
        padded = case["seqs"] * case["ctx"] * case["kv"] * case["dim"] * 8.0
        scores = 4.0 * case["seqs"] * case["heads"] * case["new"] * case["ctx"] if case["kind"] == "attend" else 0.0
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops and padded + 3 * scores < 2.5e10:
            return case


def _lens(case):
    """Tokens of every sequence in the cache and how many of them are new: the first is the longest, the others spread below."""
    n, ctx = [], []
    for b in range(case["seqs"]):
        part = (b * 37 % 64) / 128.0  # 0 .. 1/2
        ctx.append(max(1, case["ctx"] - int(case["ctx"] * part)))
        n.append(min(ctx[b], max(1, case["new"] - int(case["new"] * part))))
    return n, ctx


def work(case):
    n, ctx = _lens(case)
    held = case["dim"] * (2.0 if case["fmt"] == "bf16" else 1.0 + 1.0 / 32)  # bytes of a head row in the cache
    io = 4.0 if case["io"] == "f32" else 2.0
    if case["kind"] == "cache":  # new rows in, held, and every sequence's rows out
        rows = 2.0 * case["kv"]
        return {"bytes": rows * (sum(n) * (case["dim"] * io + held) + sum(ctx) * (held + case["dim"] * io)), "flops": 0.0}
    w = case["window"] or 1 << 40
    pairs = seen = 0
    for new, c in zip(n, ctx):
        p = c - new  # token i sees min(p + i + 1, w) keys
        full = max(0, min(new, w - p))  # tokens whose window is not yet full
        pairs += full * p + full * (full + 1) // 2 + (new - full) * w
        seen += c - max(0, p + 1 - w)
    return {"bytes": 2.0 * case["kv"] * held * seen + 4.0 * sum(n) * case["heads"] * case["dim"],
            "flops": 4.0 * case["dim"] * case["heads"] * pairs}


# --------------------------------------------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    """Queries, keys and values of all tokens, sequences one after another; keys with some channels far larger than the others,
    as a rotary projection makes them."""
    n, ctx = _lens(case)
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    kv, dim = case["kv"], case["dim"]
    loud = 0.5 + 3.0 * (torch.rand(kv, dim, generator=g, device="cuda") > 0.94) + 0.4 * torch.rand(kv, dim, generator=g, device="cuda")
    dt = DT[case["io"]]
    k = (rnd(sum(ctx), kv, dim) * loud).to(dt)
    v = (rnd(sum(ctx), kv, dim) * (0.3 + 1.4 * torch.rand(sum(ctx), kv, 1, generator=g, device="cuda"))).to(dt)
    q = rnd(sum(n), case["heads"], dim).to(dt) if case["kind"] == "attend" else None
    pages = [-(-c // PAGE) for c in ctx]
    order = torch.randperm(sum(pages), generator=g, device="cuda").int()
    table = torch.full((len(ctx), max(pages)), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(max(pages), device="cuda")[None] < torch.tensor(pages, device="cuda")[:, None]] = order
    return n, ctx, q, k, v, table, sum(pages)


def _rows_of(lens):
    """For rows of sequences one after another: which sequence, and which place in it."""
    t = torch.tensor(lens, device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), t)
    return seq, torch.arange(sum(lens), device="cuda") - (torch.cumsum(t, 0) - t)[seq]


def prepare(case, seed):
    n, ctx, q, k, v, table, pages = _inputs(case, seed)
    seq, at = _rows_of(ctx)
    fresh = at >= (torch.tensor(ctx, device="cuda") - torch.tensor(n, device="cuda"))[seq]
    keep = ~fresh if case["kind"] == "cache" else torch.ones_like(fresh)  # what the cache holds before the call
    st = dict(case=case, q=q)
    if case["kind"] == "cache":
        st["k_new"], st["v_new"] = k[fresh].contiguous(), v[fresh].contiguous()
    if own:
        from qwen3_tts_rs_amd import KVCache
        cache = KVCache(pages=pages, page_tokens=PAGE, kv_heads=case["kv"], head_dim=case["dim"], format=case["fmt"])
        held = [c - m for c, m in zip(ctx, n)] if case["kind"] == "cache" else ctx
        cache.write(0, cache.batch(held, held, table), k[keep].contiguous(), v[keep].contiguous())
        st.update(cache=cache, batch=cache.batch(n, ctx, table), whole=cache.batch(ctx, ctx, table))
        return st
    place = table[seq, at // PAGE].long() * PAGE + at % PAGE  # where each token lives
    pool = _pool(case, pages)
    _put(pool, case["fmt"], place[keep], k[keep], v[keep])
    nseq, nat = _rows_of(n)
    st.update(pool=pool, place=place, fresh=place[fresh], table=table, ctx=torch.tensor(ctx, device="cuda"),
              new=torch.tensor(n, device="cuda"), nseq=nseq, nat=nat, most_new=max(n), most_ctx=max(ctx))
    return st


# ----------------------------------------------------------------------------------------------------------- plain form
def _pool(case, pages):
    shape = (2, pages * PAGE, case["kv"], case["dim"])
    if case["fmt"] == "bf16":
        return {"codes": torch.zeros(shape, dtype=torch.bfloat16, device="cuda")}
    return {"codes": torch.zeros(shape, dtype=torch.float8_e4m3fn if case["fmt"] == "e4m3" else torch.int8, device="cuda"),
            "scale": torch.zeros(*shape[:-1], case["dim"] // 32, dtype=torch.int8, device="cuda")}


def _put(pool, fmt, place, k, v):
    x = torch.stack([k, v]).float()
    if fmt == "bf16":
        pool["codes"][:, place] = x.to(torch.bfloat16)
        return
    x = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))
    mt, et = math.frexp(TOP[fmt])
    e = (e - et + (m > mt).int()).clamp(min=-100)
    y = torch.ldexp(x, -e)
    pool["codes"][:, place] = (y.to(torch.float8_e4m3fn) if fmt == "e4m3" else y.round().to(torch.int8)).flatten(-2)
    pool["scale"][:, place] = e.squeeze(-1).to(torch.int8)


def _get(pool, fmt, place):
    codes = pool["codes"][:, place].float()
    if fmt == "bf16":
        return codes
    return torch.ldexp(codes.unflatten(-1, (-1, 32)), pool["scale"][:, place].int().unsqueeze(-1)).flatten(-2)


def run(state):
    case = state["case"]
    if own:
        cache = state["cache"]
        if case["kind"] == "cache":
            cache.write(0, state["batch"], state["k_new"], state["v_new"])
            return cache.read(0, state["whole"], dtype=DT[case["io"]])
        return cache.attend(0, state["batch"], state["q"], window=case["window"])
    fmt, dt = case["fmt"], DT[case["io"]]
    if case["kind"] == "cache":
        _put(state["pool"], fmt, state["fresh"], state["k_new"], state["v_new"])
        kv = _get(state["pool"], fmt, state["place"])
        return kv[0].to(dt), kv[1].to(dt)
    B, N, T, kv, dim = case["seqs"], state["most_new"], state["most_ctx"], case["kv"], case["dim"]
    G = case["heads"] // kv
    at = torch.arange(T, device="cuda")
    place = state["table"][:, at // PAGE].long().clamp(min=0) * PAGE + at % PAGE
    k, v = _get(state["pool"], fmt, place.flatten())  # (B T, kv, dim)
    k, v = (x.view(B, T, kv, dim).transpose(1, 2).contiguous() for x in (k, v))
    q = torch.zeros(B, N, kv, G, dim, device="cuda")
    q[state["nseq"], state["nat"]] = state["q"].float().view(-1, kv, G, dim)
    q = q.permute(0, 2, 3, 1, 4).reshape(B, kv, G * N, dim) * dim ** -0.5
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(B, kv, G, N, T)
    pos = (state["ctx"] - state["new"])[:, None] + torch.arange(N, device="cuda")  # (B, N)
    see = (at <= pos[..., None]) & (at < state["ctx"][:, None, None])
    if case["window"]:
        see = see & (at > pos[..., None] - case["window"])
    s.masked_fill_(~see[:, None, None], -math.inf)
    s -= s.amax(-1, keepdim=True).clamp(min=-3e38)
    s.exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(B, kv, G * N, T), v).view(B, kv, G, N, dim) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(B, N, kv * G, dim)
    return o[state["nseq"], state["nat"]].to(dt)


# ------------------------------------------------------------------------------------------------------ in 64 bits
def _stands_for(x, fmt):
    """What the cache gives back for rows x, in float64."""
    if fmt == "bf16":
        return x.to(torch.bfloat16).double()
    y = x.double().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    m, p = torch.frexp(y.abs().max(-1, keepdim=True).values / TOP[fmt])
    e = torch.where(m > 0.5, p, p - 1).clamp(min=-100)
    unit = torch.exp2(e.double())
    y = y / unit
    if fmt == "int8":
        y = torch.round(y)
    else:
        step = torch.exp2((torch.frexp(y)[1] - 1).clamp(min=-6).double() - 3)
        y = torch.round(y / step) * step
    return (y * unit).reshape(x.shape)


def exact(case, seed):
    n, ctx, q, k, v, _, _ = _inputs(case, seed)
    if case["kind"] == "cache":
        return _stands_for(k, case["fmt"]), _stands_for(v, case["fmt"])
    if work(case)["flops"] > 1e12:
        return None
    G = case["heads"] // case["kv"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    i = j = 0
    for new, c in zip(n, ctx):
        kd, vd = _stands_for(k[j:j + c], case["fmt"]), _stands_for(v[j:j + c], case["fmt"])
        first = torch.arange(c - new, c, device="cuda")[:, None]
        key = torch.arange(c, device="cuda")[None]
        hidden = (key > first) | (key <= first - case["window"] if case["window"] else key < 0)
        for h in range(case["heads"]):
            s = q[i:i + new, h].double() @ kd[:, h // G].T.contiguous() / math.sqrt(case["dim"])
            p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            out[i:i + new, h] = p @ vd[:, h // G].contiguous()
        i, j = i + new, j + c
    return out
