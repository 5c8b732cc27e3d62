"""The operators of a one-token decode step, as cases that can be timed and compared.

append    new K/V rows into the paged cache, rotated to their positions on the
          way, with the rotated queries (velo_cuda_kv_append)
attn      one query token per sequence over the paged cache
          (velo_cuda_decode_attention)
logprobs  log probability of given tokens, entropy and the best alternatives of
          each logits row (velo_cuda_token_logprobs)

`run` computes them in their plain form (elementary torch operations in 32
bits), or with `own` through the library; `exact` gives the same outputs from
the definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

PAGE = 16  # tokens per KV page
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ELT = {"f32": 4, "f16": 2, "bf16": 2, "int8": 1}
LARGEST = 1.2e9  # bytes of the largest listed case: a drawn one stays below

_ctx = None


def _library():
    """The library's wrapper and a context on torch's current (default) stream."""
    global _ctx
    pkg = os.path.join(os.getcwd(), "velo-core_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import velo_cuda
    if _ctx is None:
        _ctx = velo_cuda.Context(device=torch.cuda.current_device())
        _ctx.set_stream(velo_cuda.DEFAULT_STREAM)
    return velo_cuda, _ctx


# ------------------------------------------------------------------ cases

def listed():
    return [
        # a single user's short chat on a 7B-shape model (no GQA): launch latency
        dict(name="attn one short f16", op="attn", kv="f16", B=1, Hq=32, Hkv=32, D=128, lo=203, hi=203),
        # the tiny fp32 pair: one layer's decode over a prompt and its answer
        dict(name="attn tiny f32", op="attn", kv="f32", B=3, Hq=4, Hkv=4, D=64, lo=64, hi=191),
        # one user, a very long document: the split over the cache's length
        dict(name="attn one long f16", op="attn", kv="f16", B=1, Hq=64, Hkv=8, D=128, lo=100003, hi=100003),
        # the 70B-shape serving batch: 64 sequences around 4096 tokens
        dict(name="attn batch f16", op="attn", kv="f16", B=64, Hq=64, Hkv=8, D=128, lo=3900, hi=4290),
        # INT8 pages, ragged contexts of 512 to 8192 tokens
        dict(name="attn ragged int8", op="attn", kv="int8", B=128, Hq=32, Hkv=8, D=128, lo=512, hi=8192),
        # the 70B shape's decode step: one new token per sequence
        dict(name="append decode f16", op="append", kv="f16", src="f32", B=64, new_lo=1, new_hi=1, Hq=64, Hkv=8, D=128,
             ctx=1024, base=500000.0),
        # prompts of uneven lengths on the 7B shape
        dict(name="append prefill f16", op="append", kv="f16", src="f32", B=5, new_lo=701, new_hi=2577, Hq=32, Hkv=32,
             D=128, ctx=0, base=10000.0),
        # a prefill chunk into INT8 pages far into long contexts
        dict(name="append chunk int8", op="append", kv="int8", src="bf16", B=64, new_lo=17, new_hi=47, Hq=32, Hkv=8,
             D=128, ctx=512, base=10000.0),
        # the tiny fp32 pair's single token
        dict(name="append tiny f32", op="append", kv="f32", src="f32", B=1, new_lo=1, new_hi=1, Hq=4, Hkv=4, D=64,
             ctx=100, base=10000.0),
        # one sampled token of a large vocabulary with five alternatives
        dict(name="logprobs one f32", op="logprobs", src="f32", M=1, V=128256, n=5, T=1.0),
        # a verify step's rows (64 sequences x 32 nodes), scored with twenty alternatives
        dict(name="logprobs step f32", op="logprobs", src="f32", M=2048, V=128256, n=20, T=1.0),
        # rows of 64 chains of 9, 16-bit logits, at the sampling temperature
        dict(name="logprobs chains bf16", op="logprobs", src="bf16", M=576, V=32000, n=8, T=0.8),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    """One more case of the listed ones' ranges: sizes spread over their logarithm."""
    op = rng.choice(("attn", "append", "logprobs"))
    if op == "logprobs":
        src, V = rng.choice(("f32", "bf16", "f16")), _log(rng, 32, 160000)
        M = _log(rng, 1, max(1, min(4096, int(LARGEST / 2 / (V * ELT[src])))))
        return dict(op=op, src=src, M=M, V=V, n=rng.randint(1, min(20, V)), T=rng.choice((1.0, 0.7, 0.8)))
    kv = rng.choice(("f16", "f16", "int8", "f32"))
    Hq, Hkv = rng.choice(((32, 32), (64, 8), (32, 8), (4, 4), (12, 12), (8, 1), (32, 2), (40, 8), (24, 1)))
    D = rng.choice((64, 128, 128))
    if op == "attn":
        B = _log(rng, 1, 128)
        most = max(1, min(131072, int(LARGEST / 2 / (B * 2 * Hkv * D * ELT[kv]))))
        hi = _log(rng, 1, most)
        return dict(op=op, kv=kv, B=B, Hq=Hq, Hkv=Hkv, D=D, lo=rng.randint(1, hi), hi=hi)
    B = _log(rng, 1, 64)
    hi = _log(rng, 1, max(1, 12000 // B))
    return dict(op=op, kv=kv, src=rng.choice(("f32", "bf16", "f16")), B=B, new_lo=rng.randint(1, hi), new_hi=hi, Hq=Hq,
                Hkv=Hkv, D=D, ctx=_log(rng, 1, 1500), base=rng.choice((10000.0, 500000.0)))


def _spread(lo, hi, B):
    """B whole numbers from lo to hi, the same for every seed."""
    return [lo + int((hi - lo + 1) * ((0.5 + i * 0.6180339887498949) % 1.0)) for i in range(B)] if B > 1 else [hi]


def _lengths(c):
    """Cached and new tokens of each sequence."""
    if c["op"] == "attn":
        return _spread(c["lo"], c["hi"], c["B"]), [0] * c["B"]
    return _spread(max(0, c["ctx"] // 2), c["ctx"], c["B"]), _spread(c["new_lo"], c["new_hi"], c["B"])


def work(c):
    if c["op"] == "logprobs":
        return {"bytes": c["M"] * (c["V"] * ELT[c["src"]] + 12 + 8 * c["n"]), "flops": 6 * c["M"] * c["V"]}
    cached, new = _lengths(c)
    D, Hq, Hkv, B = c["D"], c["Hq"], c["Hkv"], c["B"]
    row = D * ELT[c["kv"]] + (2 if c["kv"] == "int8" else 0)  # one token's K or V of one head
    act = 4 if c["kv"] == "f32" else 2
    if c["op"] == "attn":
        pages = sum(-(-n // PAGE) for n in cached)
        return {"bytes": 2 * sum(cached) * Hkv * row + 2 * B * Hq * D * act + 4 * B * (Hq + 1) + 4 * pages,
                "flops": 4 * sum(cached) * Hq * D}
    T = sum(new)
    rows_back = 2 * T * Hkv * D * act if c["kv"] == "int8" else 0
    return {"bytes": T * (Hq + 2 * Hkv) * D * ELT[c["src"]] + T * Hq * D * act + 2 * T * Hkv * row + rows_back,
            "flops": 3 * T * (Hq + Hkv) * D}


# ------------------------------------------------------------------ inputs

def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _quantised(x):
    """INT8 rows and their f16 scales: scale = max|x| / 127, truncation."""
    m = x.abs().amax(-1)
    scale = (m / 127.0).half()
    return torch.trunc(x * (127.0 / m).unsqueeze(-1)).to(torch.int8), scale


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dev = torch.device("cuda")
    if c["op"] == "logprobs":
        M, V, n = c["M"], c["V"], c["n"]
        # every row has its own spread: from nearly certain to nearly uniform
        x = _rand(g, M, V) * (0.5 + 3.5 * torch.rand(M, 1, generator=g, device=dev))
        # every eighth row is under a grammar: nine tenths of its entries are masked out
        x[7::8] = torch.where(torch.rand(M // 8, V, generator=g, device=dev) < 0.1, x[7::8], -math.inf)
        x[7::8, V // 2] = 1.0
        s = dict(c=c, logits=x.to(DTYPES[c["src"]]),
                 tokens=torch.randint(0, V, (M,), generator=g, device=dev, dtype=torch.int32),
                 logprob=torch.empty(M, device=dev), entropy=torch.empty(M, device=dev),
                 top_tokens=torch.empty(M, n, dtype=torch.int32, device=dev), top_logprobs=torch.empty(M, n, device=dev))
        if own:
            _library()
        return s
    cached, new = _lengths(c)
    B, Hq, Hkv, D, kv = c["B"], c["Hq"], c["Hkv"], c["D"], c["kv"]
    need = [-(-(a + b) // PAGE) for a, b in zip(cached, new)]
    pages, width = sum(need), max(need)
    perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    starts = torch.tensor([sum(need[:b]) for b in range(B)], device=dev)
    col = torch.arange(width, device=dev)
    at = (starts.unsqueeze(1) + col).clamp(max=pages - 1)
    table = torch.where(col < torch.tensor(need, device=dev).unsqueeze(1), perm[at], 0).contiguous()
    pools, scales = [], [None, None]
    for i in range(2):
        x = _rand(g, pages, Hkv, PAGE, D)
        if kv == "int8":
            x, scales[i] = _quantised(x)
        pools.append(x if kv in ("f32", "int8") else x.half())
    act = torch.float32 if kv == "f32" else torch.float16
    s = dict(c=c, k_pool=pools[0], v_pool=pools[1], k_scale=scales[0], v_scale=scales[1], table=table)
    if c["op"] == "attn":
        # heads from flat to peaked
        sharp = 0.5 + 2.5 * torch.rand(1, Hq, 1, generator=g, device=dev)
        s.update(q=(_rand(g, B, Hq, D) * sharp).to(act), lens=torch.tensor(cached, dtype=torch.int32, device=dev),
                 out=torch.empty(B, Hq, D, dtype=act, device=dev), lse=torch.empty(B, Hq, device=dev))
    else:
        T = sum(new)
        # one fused projection's rows: q, k and v are slices of it
        qkv = _rand(g, T, (Hq + 2 * Hkv) * D).to(DTYPES[c["src"]])
        cut = [0]
        for n in new:
            cut.append(cut[-1] + n)
        s.update(qkv=qkv, ctx_len=torch.tensor(cached, dtype=torch.int32, device=dev),
                 seq_start=torch.tensor(cut, dtype=torch.int32, device=dev),
                 q_out=torch.empty(T, Hq, D, dtype=act, device=dev))
        q, k, v = qkv.split((Hq * D, Hkv * D, Hkv * D), 1)
        s.update(q=q.unflatten(1, (Hq, D)), k=k.unflatten(1, (Hkv, D)), v=v.unflatten(1, (Hkv, D)))
        if kv == "int8":
            s.update(k_out=torch.empty(T, Hkv, D, dtype=act, device=dev),
                     v_out=torch.empty(T, Hkv, D, dtype=act, device=dev))
    if own:
        velo_cuda, ctx = _library()
        s["cache"] = velo_cuda.KvCache(pools[0], pools[1], table, scales[0], scales[1])
        if c["op"] == "attn":
            s["workspace"] = torch.empty(ctx.decode_attention_workspace(Hq, Hkv, D), dtype=torch.uint8, device=dev)
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    if own:
        return _run_library(s)
    return {"attn": _plain_attn, "append": _plain_append, "logprobs": _plain_logprobs}[s["c"]["op"]](s)


def _run_library(s):
    c, ctx = s["c"], _ctx
    if c["op"] == "attn":
        ctx.decode_attention(s["cache"], s["q"], s["lens"], s["out"], s["workspace"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if c["op"] == "logprobs":
        ctx.token_logprobs(s["logits"], s["tokens"], s["logprob"], s["entropy"], s["top_tokens"], s["top_logprobs"],
                           temperature=c["T"])
        return {k: s[k] for k in ("logprob", "entropy", "top_tokens", "top_logprobs")}
    # one token per sequence needs no cut of the rows into sequences
    cut = None if c["new_hi"] == 1 else s["seq_start"]
    ctx.kv_append(s["cache"], s["q"], s["k"], s["v"], s["ctx_len"], s["q_out"], c["base"], seq_start=cut,
                  k_out=s.get("k_out"), v_out=s.get("v_out"))
    return _append_outputs(s, s.get("k_out"), s.get("v_out"), s["q_out"])


def _append_outputs(s, k_out, v_out, q_out):
    if s["c"]["kv"] == "int8":  # the 8-bit pages as the values they stand for: the rows just written
        return {"q": q_out, "k": k_out, "v": v_out, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    return {"q": q_out, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_attn(s):
    c = s["c"]
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]

    def rows(pool, scale):  # [B][Hkv][pages * 16][D]
        x = pool[s["table"]].float()
        if scale is not None:
            x *= scale[s["table"]].float().unsqueeze(-1)
        return x.transpose(1, 2).reshape(B, Hkv, -1, D)

    q = s["q"].float().reshape(B, Hkv, Hq // Hkv, D) / math.sqrt(D)
    x = q @ rows(s["k_pool"], s["k_scale"]).transpose(2, 3)
    seen = torch.arange(x.shape[-1], device=x.device) < s["lens"].reshape(B, 1, 1, 1)
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    z = p.sum(-1, keepdim=True)
    out = (p @ rows(s["v_pool"], s["v_scale"])) / z
    lse = (top + torch.log(z)).reshape(B, Hq)
    return {"out": out.reshape(B, Hq, D).to(s["out"].dtype), "lse": lse}


def _places(s):
    """Sequence and position of every new token."""
    t = torch.arange(s["qkv"].shape[0], device="cuda", dtype=torch.int32)
    b = (t.unsqueeze(1) >= s["seq_start"][1:]).sum(1)
    return b, (s["ctx_len"][b] + t - s["seq_start"][b]).long()


def _plain_append(s):
    c = s["c"]
    D, half = c["D"], c["D"] // 2
    b, pos = _places(s)
    # angles of far positions need 64 bits
    freq = c["base"] ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    a = pos.unsqueeze(1).double() * freq
    cos, sin = torch.cos(a).float().unsqueeze(1), torch.sin(a).float().unsqueeze(1)

    def rotated(x):
        x0, x1 = x[..., :half].float(), x[..., half:].float()
        return torch.cat((x0 * cos - x1 * sin, x0 * sin + x1 * cos), -1)

    q, k, v = rotated(s["q"]), rotated(s["k"]), s["v"].float()
    page, slot = s["table"][b, pos // PAGE].long(), pos % PAGE
    if c["kv"] != "int8":
        s["k_pool"][page, :, slot] = k.to(s["k_pool"].dtype)
        s["v_pool"][page, :, slot] = v.to(s["v_pool"].dtype)
        return _append_outputs(s, None, None, q.to(s["q_out"].dtype))
    back = []
    for x, pool, scale in ((k, s["k_pool"], s["k_scale"]), (v, s["v_pool"], s["v_scale"])):
        ints, sc = _quantised(x)
        pool[page, :, slot] = ints
        scale[page, :, slot] = sc
        back.append((ints.float() * sc.float().unsqueeze(-1)).half())
    return _append_outputs(s, back[0], back[1], q.to(s["q_out"].dtype))


def _plain_logprobs(s):
    c, n = s["c"], s["c"]["n"]
    x = s["logits"].float()
    # the order of values as whole numbers, the lower index above among equal ones
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32
    key += torch.arange(c["V"] - 1, -1, -1, device="cuda")
    top = (c["V"] - 1 - (torch.topk(key, n, sorted=True).values & 0xFFFFFFFF)).int()
    x = x * (1.0 / c["T"])
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    z = e.sum(-1)
    log_z = torch.log(z)
    logprob = torch.gather(d, 1, s["tokens"].long().unsqueeze(1)).squeeze(1) - log_z
    entropy = log_z - torch.where(e > 0, e * d, 0.0).sum(-1) / z
    return {"logprob": logprob, "entropy": entropy, "top_tokens": top,
            "top_logprobs": torch.gather(d, 1, top.long()) - log_z.unsqueeze(1)}


# ------------------------------------------------------------------ in 64 bits

def exact(c, seed):
    s = prepare(c, seed)
    return {"attn": _exact_attn, "append": _exact_append, "logprobs": _exact_logprobs}[c["op"]](s)


def _exact_attn(s):
    c, outs, lses = s["c"], [], []
    group = c["Hq"] // c["Hkv"]
    for b, n in enumerate(s["lens"].tolist()):  # a sequence at a time
        ids = s["table"][b, :-(-n // PAGE)].long()
        kv = []
        for pool, scale in ((s["k_pool"], s["k_scale"]), (s["v_pool"], s["v_scale"])):
            x = pool[ids].double()
            if scale is not None:
                x = x * scale[ids].double()[..., None]
            x = x.permute(0, 2, 1, 3).reshape(-1, c["Hkv"], c["D"])[:n]
            kv.append(x.permute(1, 0, 2).repeat_interleave(group, 0))  # [Hq][n][D]
        logits = (kv[0] * s["q"][b].double()[:, None, :]).sum(-1) / math.sqrt(c["D"])
        lse = torch.logsumexp(logits, -1)
        outs.append((torch.exp(logits - lse[:, None])[..., None] * kv[1]).sum(1))
        lses.append(lse)
    return {"out": torch.stack(outs), "lse": torch.stack(lses)}


def _exact_append(s):
    c = s["c"]
    half = c["D"] // 2
    seq = torch.repeat_interleave(torch.arange(c["B"], device="cuda"), s["seq_start"].diff().long())
    step = torch.arange(seq.numel(), device="cuda") - s["seq_start"].long()[seq]
    pos = s["ctx_len"].long()[seq] + step
    turn = torch.exp(-math.log(c["base"]) * 2 * torch.arange(half, device="cuda", dtype=torch.float64) / c["D"])
    rot = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos.double()[:, None] * turn)[:, None]

    def turned(x):
        y = torch.complex(x[..., :half].double(), x[..., half:].double()) * rot
        return torch.cat((y.real, y.imag), -1)

    page, slot = s["table"].long()[seq, torch.div(pos, PAGE, rounding_mode="floor")], pos % PAGE
    res = {"q": turned(s["q"])}
    for name, x in (("k", turned(s["k"])), ("v", s["v"].double())):
        if c["kv"] == "int8":
            m = x.abs().max(-1).values
            sc = s[name + "_scale"].double()
            sc[page, :, slot] = m / 127
            res[name + "_scale"] = sc
            res[name] = torch.trunc(x * 127 / m[..., None]) * (m / 127).half().double()[..., None]
        else:
            pool = s[name + "_pool"].double()
            pool[page, :, slot] = x
            res[name + "_pool"] = pool
    return res


def _exact_logprobs(s):
    c, res = s["c"], {k: [] for k in ("logprob", "entropy", "top_tokens", "top_logprobs")}
    for part, tok in zip(s["logits"].split(64), s["tokens"].long().split(64)):  # some rows at a time
        x = part.double() / c["T"]
        lp = x - torch.logsumexp(x, -1, keepdim=True)
        best = torch.sort(part.double(), dim=-1, descending=True, stable=True).indices[:, :c["n"]]
        res["logprob"].append(lp.gather(1, tok[:, None])[:, 0])
        res["entropy"].append(torch.special.entr(lp.exp()).sum(-1))
        res["top_tokens"].append(best.int())
        res["top_logprobs"].append(lp.gather(1, best))
    return {k: torch.cat(v) for k, v in res.items()}
