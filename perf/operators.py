"""Paged-cache operators: what each computes in its plain form, and the sizes they are timed at.

Three operators that a layer of a served Llama-family model runs one after another over one
paged key-value cache (pages of `page` slots, [pages, kv heads, page, head dim]; sequence b's
token t is in slot t % page of page page_table[b, t // page]):

  rope    norms of queries and keys for each head, rotation by position, append to the cache
  decode  attention of one new token per sequence over the cache
  prompt  attention of prompt chunks (the newest tokens of each sequence) over the cache

Position p sees key j when j <= p and, with a window, p - j < window or j < sinks.
"""

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
THETA = 500000.0


def _case(name, op, dtype, hd, nq, nkv, page, batch, ctx_lo, ctx_hi, new_lo=1, new_hi=1, window=0, sinks=0,
          tables="fp32", packed=False, norm=True):
    return {"name": name, "op": op, "dtype": dtype, "hd": hd, "nq": nq, "nkv": nkv, "page": page, "batch": batch,
            "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "new_lo": new_lo, "new_hi": new_hi, "window": window, "sinks": sinks,
            "tables": tables, "packed": packed, "norm": norm}


def listed():
    return [
        # one user's chat, one step of the 8B heads: latency is all there is
        _case("rope-step-1", "rope", "fp16", 128, 32, 8, 16, 1, 517, 517, packed=True, tables="fp16"),
        # a decode batch of the 1B heads
        _case("rope-step-192", "rope", "bf16", 64, 32, 8, 32, 192, 9, 1021),
        # several prompts of odd lengths in one pass, 70B heads, q|k|v side by side as one GEMM leaves them
        _case("rope-prompts-ragged", "rope", "bf16", 128, 64, 8, 64, 7, 301, 4099, 301, 4099, packed=True),
        # one user's chat, a short context
        _case("decode-1-short", "decode", "fp16", 128, 32, 8, 16, 1, 517, 517),
        # one user over a whole book: only the cache's length gives parallel work
        _case("decode-1-long", "decode", "bf16", 128, 32, 8, 64, 1, 131071, 131071),
        # a serving batch whose sequences differ by two orders of magnitude
        _case("decode-64-ragged", "decode", "fp16", 128, 32, 8, 16, 64, 131, 16384),
        # long chats held by a window and four sinks, 1B heads
        _case("decode-160-window", "decode", "bf16", 64, 32, 8, 32, 160, 700, 30011, window=1024, sinks=4),
        # one short odd prompt, 1B heads
        _case("prompt-1-short", "prompt", "fp16", 64, 32, 8, 16, 1, 257, 257, 257, 257),
        # one whole long prompt, 8B heads
        _case("prompt-1-8k", "prompt", "fp16", 128, 32, 8, 64, 1, 8192, 8192, 8192, 8192),
        # a chunk of a prompt far into its context: few rows, a long cache
        _case("prompt-chunk-deep", "prompt", "bf16", 128, 32, 8, 16, 1, 32005, 32005, 256, 256),
        # several prompts of odd lengths, some with a cached prefix
        _case("prompt-6-ragged", "prompt", "bf16", 128, 32, 8, 32, 6, 777, 5003, 129, 2111),
        # a long prompt under a window with sinks, 70B heads
        _case("prompt-1-window", "prompt", "bf16", 128, 64, 8, 128, 1, 16001, 16001, 16001, 16001, window=4096,
              sinks=4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "decode", "prompt"])
    hd = rng.choice([64, 128])
    nkv = rng.choice([1, 2, 4, 8])
    nq = nkv * rng.choice([1, 2, 3, 4, 5, 8] if op != "decode" else [1, 2, 4, 6, 8, 12])
    dtype = rng.choice(["fp16", "bf16"])
    page = rng.choice([16, 32, 64, 128, 256])
    window, sinks = 0, 0
    if op != "rope" and rng.random() < 0.5:
        window, sinks = _log_int(rng, 16, 4096), rng.choice([0, 1, 4, 64])
    if op == "rope":
        batch = _log_int(rng, 1, 200)
        if rng.random() < 0.5:
            lo, hi, n_lo, n_hi = 1, _log_int(rng, 16, 4096), 1, 1
        else:
            n_hi = max(1, _log_int(rng, 16, 16384) // batch)
            n_lo = max(1, n_hi // 9)
            lo, hi = n_lo, n_hi
    elif op == "decode":
        batch = _log_int(rng, 1, 200)
        hi = max(1, min(131072, _log_int(rng, 64, 131072), 262144 // batch))
        lo, n_lo, n_hi = max(1, hi // rng.choice([1, 3, 100])), 1, 1
    else:
        batch = _log_int(rng, 1, 16)
        n_hi = max(1, _log_int(rng, 33, 8192) // batch)
        n_lo = max(1, n_hi // rng.choice([1, 7]))
        past = rng.choice([0, 0, _log_int(rng, 16, 8192) // batch])
        lo, hi = n_lo + past, n_hi + past
    return _case("", op, dtype, hd, nq, nkv, page, batch, lo, hi, n_lo, n_hi, window, sinks,
                 tables=rng.choice(["fp32", dtype]), packed=rng.random() < 0.5,
                 norm=rng.random() < 0.8)


def _spread(lo, hi, n, turn):
    """n whole numbers from lo to hi, even in their logarithm, in a mixed order."""
    if n == 1:
        return [hi]
    vals = [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]
    step = next(s for s in range(max(1, int(n * 0.618)) + turn, 3 * n + 7) if math.gcd(s, n) == 1)
    return [vals[(i * step) % n] for i in range(n)]


def _lengths(case):
    """(tokens in the cache with the new ones, new tokens) of every sequence."""
    kv = _spread(case["ctx_lo"], case["ctx_hi"], case["batch"], 0)
    if case["new_hi"] == 1:
        return kv, [1] * case["batch"]
    if (case["new_lo"], case["new_hi"]) == (case["ctx_lo"], case["ctx_hi"]):
        return kv, list(kv)
    new = _spread(case["new_lo"], case["new_hi"], case["batch"], 1)
    return [max(a, b) for a, b in zip(kv, new)], new


def prepare(case, seed):
    dev = torch.device("cuda")
    dt, hd, nq, nkv, page = DTYPES[case["dtype"]], case["hd"], case["nq"], case["nkv"], case["page"]
    kv, new = _lengths(case)
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32 if math.prod(shape) < 1 << 26 else dt)

    need = [-(-n // page) for n in kv]
    n_pages = sum(need) + 3          # a pool with a few free pages
    order = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32)
    table = torch.full((len(kv), max(need)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    T = offsets[-1]
    s = {"case": case, "kv": kv, "new": new, "offsets": offsets, "scale": hd ** -0.5,
         "k_pages": normal(n_pages, nkv, page, hd).to(dt), "v_pages": normal(n_pages, nkv, page, hd).to(dt),
         "page_table": table, "kv_lens": torch.tensor(kv, dtype=torch.int32, device=dev),
         "q_offsets": None if case["new_hi"] == 1 else torch.tensor(offsets, dtype=torch.int32, device=dev)}
    if case["op"] != "rope":
        # queries that make some keys stand out, as trained heads do
        s["q"] = (normal(T, nq, hd).float() * 1.7).to(dt)
        return s
    if case["packed"]:
        qkv = (normal(T, nq + 2 * nkv, hd).float() * 1.3).to(dt)
        s["q"], s["k"], s["v"] = qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:]
    else:
        for name, n in (("q", nq), ("k", nkv), ("v", nkv)):
            s[name] = (normal(T, n, hd).float() * 1.3).to(dt)
    s["q_weight"] = (1 + 0.1 * normal(hd)).to(dt) if case["norm"] else None
    s["k_weight"] = (1 + 0.1 * normal(hd)).to(dt) if case["norm"] else None
    inv = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=dev) / hd)
    ang = torch.arange(max(kv), dtype=torch.float64, device=dev)[:, None] * inv
    ang = torch.cat([ang, ang], dim=-1)
    tt = DTYPES.get(case["tables"], torch.float32)
    s["cos"], s["sin"] = ang.cos().to(tt), ang.sin().to(tt)
    return s


# ------------------------------------------------------------------ plain forms

def _plain_head(x, weight, cos, sin):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    h = x.shape[-1] // 2
    turned = torch.cat([-x[..., h:], x[..., :h]], dim=-1)
    return x * cos + turned * sin


def _plain_rope(s):
    dt, page = s["q"].dtype, s["case"]["page"]
    q_offsets = s["q_offsets"]
    T, B = s["q"].shape[0], len(s["kv"])
    rows = torch.arange(T, device=s["q"].device)
    if q_offsets is None:
        seq, pos = rows, s["kv_lens"].long() - 1
    else:
        seq = torch.searchsorted(q_offsets[1:].long(), rows, right=True).clamp_(max=B - 1)
        pos = s["kv_lens"].long()[seq] - q_offsets.long()[seq + 1] + rows
    cos, sin = s["cos"][pos][:, None].float(), s["sin"][pos][:, None].float()
    q = _plain_head(s["q"], s["q_weight"], cos, sin).to(dt)
    k = _plain_head(s["k"], s["k_weight"], cos, sin).to(dt)
    pages = s["page_table"][seq, pos // page].long()
    s["k_pages"][pages, :, pos % page] = k
    s["v_pages"][pages, :, pos % page] = s["v"]
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _tokens(pool, table_row, n, page):
    """The first n tokens of one sequence, [kv heads, n, head dim] in 32 bits."""
    got = pool[table_row[:-(-n // page)].long()].float()
    return got.transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, :n]


def _plain_attend(q, k, v, first, window, sinks, scale):
    """q [n, nq, hd] at positions first.. over k, v [nkv, m, hd]; all in 32 bits."""
    n, nq, hd = q.shape
    nkv, m, _ = k.shape
    group = nq // nkv
    out = torch.empty_like(q)
    step = max(1, min(1024, (1 << 28) // (nq * max(1, min(m, window + sinks + 1024 if window else m)))))
    for a in range(0, n, step):
        e = min(n, a + step)
        lo = max(0, first + a - window + 1) if window else 0
        hi = first + e
        keep = min(sinks, lo)
        kk = torch.cat([k[:, :keep], k[:, lo:hi]], dim=1) if keep else k[:, lo:hi]
        vv = torch.cat([v[:, :keep], v[:, lo:hi]], dim=1) if keep else v[:, lo:hi]
        j = torch.cat([torch.arange(keep, device=q.device), torch.arange(lo, hi, device=q.device)])
        p = torch.arange(first + a, first + e, device=q.device)[:, None]
        hidden = j > p
        if window:
            hidden |= (p - j >= window) & (j >= sinks)
        qq = q[a:e].reshape(e - a, nkv, group, hd).permute(1, 2, 0, 3).reshape(nkv, group * (e - a), hd)
        x = torch.matmul(qq, kk.transpose(1, 2)).mul_(scale).view(nkv, group, e - a, -1)
        x.masked_fill_(hidden, -math.inf)
        x = torch.exp(x.sub_(x.max(-1, keepdim=True).values))
        total = x.sum(-1, keepdim=True)
        o = torch.matmul(x.view(nkv, group * (e - a), -1), vv).view(nkv, group, e - a, hd) / total
        out[a:e] = o.permute(2, 0, 1, 3).reshape(e - a, nq, hd)
    return out


def _plain_attention(s):
    c = s["case"]
    out = torch.empty_like(s["q"])
    for b, (n, m) in enumerate(zip(s["kv"], s["new"])):
        a, e = s["offsets"][b], s["offsets"][b + 1]
        k = _tokens(s["k_pages"], s["page_table"][b], n, c["page"])
        v = _tokens(s["v_pages"], s["page_table"][b], n, c["page"])
        out[a:e] = _plain_attend(s["q"][a:e].float(), k, v, n - m, c["window"], c["sinks"], s["scale"]).to(out.dtype)
    return out


def run(s):
    op = s["case"]["op"]
    if not own:
        return _plain_rope(s) if op == "rope" else _plain_attention(s)
    from liteweight_b200 import kernels
    cache = (s["k_pages"], s["v_pages"], s["page_table"], s["kv_lens"])
    if op == "rope":
        q = kernels.qk_norm_rope(s["q"], s["k"], s["v"], s["cos"], s["sin"], *cache, s["q_offsets"],
                                 q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS)
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    window, sinks = s["case"]["window"] or None, s["case"]["sinks"]
    if op == "decode":
        return kernels.paged_attention(s["q"], *cache, window=window, sinks=sinks, scale=s["scale"])
    return kernels.prompt_attention(s["q"], *cache, s["q_offsets"], window=window, sinks=sinks, scale=s["scale"])


# ------------------------------------------------------------------ the same from the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    hd, page, group = case["hd"], case["page"], case["nq"] // case["nkv"]
    dev = s["q"].device
    if case["op"] == "rope":
        pos = torch.cat([torch.arange(n - m, n, device=dev) for n, m in zip(s["kv"], s["new"])])
        seq = torch.cat([torch.full((m,), b, device=dev) for b, m in enumerate(s["new"])])
        c, si = s["cos"].double()[pos].unsqueeze(1), s["sin"].double()[pos].unsqueeze(1)

        def head(x, w):
            x = x.double()
            if w is not None:
                x = x / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
            y = x * c
            y[..., :hd // 2] -= x[..., hd // 2:] * si[..., :hd // 2]
            y[..., hd // 2:] += x[..., :hd // 2] * si[..., hd // 2:]
            return y

        pools = {}
        for name, new in (("k", head(s["k"], s["k_weight"])), ("v", s["v"].double())):
            flat = s[name + "_pages"].double().transpose(1, 2).reshape(-1, case["nkv"], hd)
            flat[s["page_table"][seq, pos // page].long() * page + pos % page] = new
            pools[name] = flat.view(-1, page, case["nkv"], hd).transpose(1, 2)
        return {"q": head(s["q"], s["q_weight"]), "k_pages": pools["k"], "v_pages": pools["v"]}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    for b, (n, m) in enumerate(zip(s["kv"], s["new"])):
        t = torch.arange(n, device=dev)
        page_of, slot = s["page_table"][b].long()[t // page], t % page
        rows = max(1, min(m, (1 << 25) // n))
        for h in range(case["nkv"]):
            k, v = s["k_pages"][page_of, h, slot].double(), s["v_pages"][page_of, h, slot].double()
            for a in range(0, m, rows):
                e = min(m, a + rows)
                p = torch.arange(n - m + a, n - m + e, device=dev).view(-1, 1)
                seen = t <= p
                if case["window"]:
                    seen &= (t > p - case["window"]) | (t < case["sinks"])
                for i in range(h * group, (h + 1) * group):
                    x = s["q"][s["offsets"][b] + a:s["offsets"][b] + e, i].double() @ k.T * s["scale"]
                    w = torch.softmax(torch.where(seen, x, -math.inf), dim=-1)
                    out[s["offsets"][b] + a:s["offsets"][b] + e, i] = w @ v
    return out


def work(case):
    kv, new = _lengths(case)
    hd, nq, nkv, window, sinks = case["hd"], case["nq"], case["nkv"], case["window"], case["sinks"]
    T = sum(new)
    if case["op"] == "rope":
        el = 4 if case["tables"] == "fp32" else 2
        distinct = len({p for n, m in zip(kv, new) for p in range(n - m, n)})
        return {"bytes": 2 * 2 * T * (nq + 2 * nkv) * hd + 2 * distinct * hd * el, "flops": T * (nq + nkv) * hd * 7}
    pairs = keys = 0
    for n, m in zip(kv, new):
        first = n - m
        if not window:
            pairs += m * first + m * (m + 1) // 2
            keys += n
            continue
        for p in range(first, n):
            lo = max(0, p - window + 1)
            pairs += p + 1 - lo + min(sinks, lo)
        lo = max(0, first - window + 1)
        keys += n - lo + min(sinks, lo)
    return {"bytes": 2 * (2 * T * nq * hd + 2 * keys * nkv * hd), "flops": 4 * pairs * nq * hd}
