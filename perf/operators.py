"""Performance cases of four operators of a quantised decode step.

  int4     a linear with 4-bit weights and one scale per group of inputs, from one
           token to a prompt
  append   q / k norm, RoPE and the new K/V into pages held in 8 bits with one scale
           per token and head; the touched pages are read back as the values they hold
  attn     decode attention of a batch over such pages
  sample   tokens drawn from logits with temperature, top-k, top-p and min-p

The plain forms are elementary torch operations in fp32 (fp64 for the angles of RoPE
and for the masses of the sampled distribution, whose borders decide a token).
`exact` is each operator's definition in fp64.
"""
import math

import numpy as np
import torch

own = False

# hidden, q heads, kv heads, head dim, FFN width of the supported model shapes
SHAPES = [(4096, 32, 8, 128, 12288), (5120, 40, 8, 128, 17408), (5120, 64, 8, 128, 25600)]
# q heads, kv heads, head dim
HEADS = [(32, 8, 128), (40, 8, 128), (64, 8, 128), (16, 8, 64), (32, 32, 64), (16, 1, 128)]
EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # the smallest call: one token through one 4096 x 4096 projection
        {"name": "int4_1_token", "kind": "int4", "m": 1, "k": 4096, "n": 4096, "gs": 128, "bias": False},
        # single-stream decode: gate and up projections of one token as one matrix
        {"name": "int4_1_token_gate_up", "kind": "int4", "m": 1, "k": 5120, "n": 34816, "gs": 128, "bias": False},
        # batched decode: twelve sequences through a down projection, fine groups
        {"name": "int4_12_tokens_down", "kind": "int4", "m": 12, "k": 12288, "n": 4096, "gs": 64, "bias": False},
        # a prompt of odd length through a gate projection
        {"name": "int4_prompt_1500", "kind": "int4", "m": 1500, "k": 4096, "n": 12288, "gs": 128, "bias": True},
        # one new token of each sequence of a batch, far into its context
        {"name": "append_batch_16", "kind": "append", "n": 16, "prompt": False, "hq": 32, "hkv": 8, "d": 128,
         "page": 16, "first": 90000},
        # a whole prompt of one sequence, continuing a half-filled page
        {"name": "append_prompt_2000", "kind": "append", "n": 2000, "prompt": True, "hq": 40, "hkv": 8, "d": 128,
         "page": 16, "first": 1003},
        # a few short chats: latency counts
        {"name": "attn_short", "kind": "attn", "b": 4, "hq": 16, "hkv": 8, "d": 64, "page": 32, "ctx": 700,
         "ragged": True},
        # single-stream decode, long context
        {"name": "attn_16k", "kind": "attn", "b": 1, "hq": 32, "hkv": 8, "d": 128, "page": 16, "ctx": 16384,
         "ragged": False},
        # a serving batch of different lengths
        {"name": "attn_batch", "kind": "attn", "b": 16, "hq": 40, "hkv": 8, "d": 128, "page": 16, "ctx": 12000,
         "ragged": True},
        # single-stream sampling with the usual filters
        {"name": "sample_1", "kind": "sample", "m": 1, "v": 151936, "mixed": False, "t": 0.7, "top_k": 20,
         "top_p": 0.8, "min_p": 0.0},
        # a batch whose requests each bring their own settings
        {"name": "sample_16_mixed", "kind": "sample", "m": 16, "v": 151936, "mixed": True},
        # a wide batch over an odd vocabulary, min-p at a high temperature
        {"name": "sample_64", "kind": "sample", "m": 64, "v": 50257, "mixed": False, "t": 1.3, "top_k": 0,
         "top_p": 1.0, "min_p": 0.05},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["int4", "append", "attn", "sample"])
    if kind == "int4":
        h, hq, hkv, d, f = rng.choice(SHAPES)
        k, n = rng.choice([(h, (hq + 2 * hkv) * d), (hq * d, h), (h, f), (f, h), (1024, 4096)])
        if rng.random() < 0.3:                       # odd sizes
            n = max(1, n - rng.randrange(1, 200))
            k -= 32 * rng.randrange(0, 8)
        gs = rng.choice([g for g in (128, 128, 64, 32) if k % g == 0])
        m = _log_int(rng, 1, min(2048, max(1, 1500 * 4096 * 12288 // (n * k))))
        if rng.random() < 0.5:                       # decode rather than a prompt
            m = rng.randrange(1, 17)
        return {"kind": kind, "m": m, "k": k, "n": n, "gs": gs, "bias": rng.random() < 0.3}
    if kind == "append":
        hq, hkv, d = rng.choice(HEADS[:4])
        prompt = rng.random() < 0.5
        return {"kind": kind, "n": _log_int(rng, 2, 2000) if prompt else rng.randrange(1, 17), "prompt": prompt,
                "hq": hq, "hkv": hkv, "d": d, "page": rng.choice([16, 16, 32, 64]),
                "first": _log_int(rng, 1, 100000) - 1}
    if kind == "attn":
        hq, hkv, d = rng.choice(HEADS)
        b = _log_int(rng, 1, 16)
        return {"kind": kind, "b": b, "hq": hq, "hkv": hkv, "d": d, "page": rng.choice([16, 16, 32, 64]),
                "ctx": _log_int(rng, 1, min(16384, 16 * 12000 * 8 // (b * hkv))),
                "ragged": b > 1 and rng.random() < 0.7}
    v = rng.choice([32000, 50257, 151936, rng.randrange(1000, 152000)])
    m = _log_int(rng, 1, 32)
    if rng.random() < 0.4:
        return {"kind": kind, "m": m, "v": v, "mixed": True}
    return {"kind": kind, "m": m, "v": v, "mixed": False, "t": round(rng.uniform(0.3, 1.6), 2),
            "top_k": rng.choice([0, _log_int(rng, 1, 1000)]), "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.99), 2)]),
            "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.2), 2)])}


# ── inputs ───────────────────────────────────────────────────────────────────

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).half()


def _norm_w(g, n):
    return (1.0 + 0.1 * torch.randn(n, generator=g, device="cuda")).half()


def _q8_pages(g, slots, hkv, page, d):
    """Pages of 8-bit K and V and their scales, holding values of about N(0, 1):
    codes [slots, Hkv, P, D] (V stored with the tokens of a dim adjacent), scales
    [slots, Hkv, P]."""
    def codes(*shape):
        return (torch.randn(*shape, generator=g, device="cuda") * 44.0).round_().clamp_(-127, 127).to(torch.int8)

    def scales():
        return ((0.8 + 0.4 * torch.rand(slots, hkv, page, generator=g, device="cuda")) / 44.0).half()
    return codes(slots, hkv, page, d), codes(slots, hkv, d, page).transpose(-1, -2), scales(), scales()


def _lengths(g, case):
    """Tokens of each item: all of them `ctx`, or spread down to a sixteenth of it."""
    b, ctx = case["b"], case["ctx"]
    if not case["ragged"]:
        return torch.full((b,), ctx, dtype=torch.int32, device="cuda")
    n = (ctx * torch.exp(-math.log(16.0) * torch.rand(b, generator=g, device="cuda"))).int().clamp_(1)
    n[0] = ctx
    return n


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    st = {"case": case}
    if kind == "int4":
        n, k, gs = case["n"], case["k"], case["gs"]
        st["x"] = _normal(g, case["m"], k)
        st["codes"] = (torch.randn(n, k, generator=g, device="cuda") * 2.8).round_().clamp_(-8, 7).to(torch.int8)
        st["scale"] = ((0.75 + 0.5 * torch.rand(n, k // gs, generator=g, device="cuda")) * (0.02 / 2.8)).half()
        st["bias"] = _normal(g, n, std=0.5) if case["bias"] else None
        if own:   # a program lays its weights out once, when it loads them
            from helm_amd.kernels import Int4Weight
            st["weight"] = Int4Weight.pack(st["codes"], st["scale"])
        return st
    if kind == "append":
        n, hq, hkv, d, page = case["n"], case["hq"], case["hkv"], case["d"], case["page"]
        if case["prompt"]:
            pos = case["first"] + torch.arange(n, device="cuda")
            local = pos // page - case["first"] // page
            n_pages = int(case["first"] + n - 1) // page - case["first"] // page + 1
        else:
            pos = case["first"] + torch.randint(0, 5 * page, (n,), generator=g, device="cuda")
            local, n_pages = torch.arange(n, device="cuda"), n
        order = torch.randperm(n_pages, generator=g, device="cuda").int()
        st["qkv"] = _normal(g, n, (hq + 2 * hkv) * d)
        st["q_norm"], st["k_norm"] = _norm_w(g, d), _norm_w(g, d)
        st["positions"], st["offsets"] = pos.int(), (pos % page).int()
        st["slots"] = order[local].contiguous()
        st["inv_freq"] = (1.0 / THETA ** (torch.arange(0, d, 2, device="cuda").double() / d)).float()
        st["pages"] = order
        st["pool"] = _q8_pages(g, n_pages, hkv, page, d)
        st["q_out"] = torch.empty(n, hq, d, dtype=torch.float16, device="cuda")
        if own:   # the view of its pool that a program keeps
            from helm_amd.kernels import attention as ka
            st["view"] = ka.Q8PoolView.of_pool(*st["pool"])
        return st
    if kind == "attn":
        hkv, d, page = case["hkv"], case["d"], case["page"]
        n = _lengths(g, case)
        cols = -(-case["ctx"] // page)
        order = torch.randperm(case["b"] * cols, generator=g, device="cuda").int()
        st["q"] = _normal(g, case["b"], case["hq"], d)
        st["pool"] = _q8_pages(g, case["b"] * cols, hkv, page, d)
        st["page_table"], st["seq_lens"] = order.view(case["b"], cols), n
        if own:   # the view of its pool and the split workspace that a decode loop keeps
            from helm_amd.kernels import attention as ka
            st["view"] = ka.Q8PoolView.of_pool(*st["pool"])
            st["workspace"] = ka.AttnWorkspace(st["q"].device)
        return st
    m, v = case["m"], case["v"]
    x = torch.randn(m, v, generator=g, device="cuda") * 2.5
    x += 9.0 * (torch.rand(m, v, generator=g, device="cuda") < 20.0 / v) * torch.rand(m, v, generator=g, device="cuda")
    st["logits"] = x.half()
    st["u"] = torch.rand(m, generator=g, device="cuda")
    if case["mixed"]:
        def pick(values, dtype):
            i = torch.randint(0, len(values), (m,), generator=g, device="cuda")
            return torch.tensor(values, dtype=dtype, device="cuda")[i]
        st["temperature"] = pick([0.0, 0.3, 0.7, 1.0, 1.0, 1.5], torch.float32)
        st["top_k"] = pick([0, 0, 1, 20, 50, 400], torch.int32)
        st["top_p"] = pick([1.0, 0.5, 0.8, 0.9, 0.95], torch.float32)
        st["min_p"] = pick([0.0, 0.0, 0.02, 0.1], torch.float32)
    else:
        st["temperature"], st["top_k"] = case["t"], case["top_k"]
        st["top_p"], st["min_p"] = case["top_p"], case["min_p"]
    if own:       # the workspace that a decode loop keeps
        from helm_amd.kernels import fused
        st["workspace"] = fused.sample_workspace(m, v, x.device)
    return st


# ── one pass ─────────────────────────────────────────────────────────────────

def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    from helm_amd.kernels import attention as ka
    from helm_amd.kernels import fused, int4_linear

    case, kind = st["case"], st["case"]["kind"]
    if kind == "int4":
        return int4_linear(st["x"], st["weight"], st["bias"])
    if kind == "append":
        q = fused.qk_norm_rope_append_q8(st["qkv"], st["q_norm"], st["k_norm"], EPS, st["positions"], st["inv_freq"],
                                         st["q_out"], st["view"], st["slots"], st["offsets"], case["hq"],
                                         case["hkv"], case["d"], case["page"])
        held = ka.dequantize_pages(st["view"], st["pages"])
        return q, held.k, held.v
    if kind == "attn":
        return ka.paged_decode_attention_q8(st["q"], st["view"], st["page_table"], st["seq_lens"], case["page"],
                                            workspace=st["workspace"])
    return fused.sample(st["logits"], st["u"], st["temperature"], st["top_k"], st["top_p"], st["min_p"],
                        workspace=st["workspace"])


def _run_plain(st):
    return {"int4": _int4, "append": _append, "attn": _attn, "sample": _sample}[st["case"]["kind"]](st)


def _int4(st):
    n, k, gs = st["case"]["n"], st["case"]["k"], st["case"]["gs"]
    w = (st["codes"].float().view(n, k // gs, gs) * st["scale"].float()[:, :, None]).view(n, k)
    y = torch.matmul(st["x"].float(), w.t())
    if st["bias"] is not None:
        y = y + st["bias"].float()
    return y.half()


def _quantise(x):
    s = (x.abs().amax(-1) / 127.0).half()
    div = torch.where(s > 0, s, torch.ones_like(s)).float()
    c = torch.where(s[..., None] > 0, torch.round(x / div[..., None]).clamp(-127, 127), torch.zeros_like(x))
    return c.to(torch.int8), s


def _append(st):
    case = st["case"]
    n, hq, hkv, d = case["n"], case["hq"], case["hkv"], case["d"]
    x = st["qkv"].float().view(n, hq + 2 * hkv, d)
    qk, v = x[:, :hq + hkv], x[:, hq + hkv:]
    w = torch.cat([st["q_norm"].float().expand(hq, d), st["k_norm"].float().expand(hkv, d)])
    qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS) * w
    ang = st["positions"].double()[:, None] * st["inv_freq"].double()
    c = torch.cat([ang.cos(), ang.cos()], -1).float()[:, None]
    s = torch.cat([ang.sin(), ang.sin()], -1).float()[:, None]
    qk = qk * c + torch.cat([-qk[..., d // 2:], qk[..., :d // 2]], -1) * s
    k_pool, v_pool, k_scale, v_scale = st["pool"]
    slots, offs = st["slots"].long(), st["offsets"].long()
    k_pool[slots, :, offs], k_scale[slots, :, offs] = _quantise(qk[:, hq:])
    v_pool[slots, :, offs], v_scale[slots, :, offs] = _quantise(v)
    pages = st["pages"].long()
    return (qk[:, :hq].half(), (k_pool[pages].float() * k_scale[pages].float()[..., None]).half(),
            (v_pool[pages].float() * v_scale[pages].float()[..., None]).half())


def _gathered(codes, scales, table):
    """fp32 [B, Hkv, tokens, D] of the pages of a table [B, pages]."""
    x = codes[table].float() * scales[table].float()[..., None]
    b, c, h, p, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, c * p, d)


def _attn(st):
    case = st["case"]
    b, hq, hkv, d = case["b"], case["hq"], case["hkv"], case["d"]
    k_pool, v_pool, k_scale, v_scale = st["pool"]
    table = st["page_table"].long()
    k, v = _gathered(k_pool, k_scale, table), _gathered(v_pool, v_scale, table)
    q = st["q"].float().view(b, hkv, hq // hkv, d)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(d)
    live = torch.arange(k.shape[2], device="cuda") < st["seq_lens"][:, None]
    s = s.masked_fill(~live[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).view(b, hq, d).half()


def _per_row(x, m, dtype):
    return (x if torch.is_tensor(x) else torch.full((m,), x, device="cuda")).to(dtype)[:, None]


def _sample(st):
    logits, u = st["logits"], st["u"].double()[:, None]
    m, v = logits.shape
    t, k = _per_row(st["temperature"], m, torch.float64), _per_row(st["top_k"], m, torch.int64)
    # (filters and temperatures are fp32 numbers, whichever way they are given)
    p, low = (_per_row(st[n], m, torch.float32).double() for n in ("top_p", "min_p"))
    t = t.float().double()
    ranked, index = torch.sort(logits.float(), dim=-1, descending=True, stable=True)
    z = (ranked.double() - ranked[:, :1].double()) / torch.where(t > 0, t, torch.ones_like(t))
    w = torch.exp(z)
    rank = torch.arange(v, device="cuda")
    w = torch.where((k <= 0) | (rank < k), w, torch.zeros_like(w))
    cum = torch.cumsum(w, -1)
    stays = ((p >= 1) | (cum - w < p * cum[:, -1:])) & (w >= low)
    stays[:, 0] = True
    w = torch.where(stays, w, torch.zeros_like(w))
    cum = torch.cumsum(torch.zeros_like(w).scatter_(-1, index, w), -1)
    token = (cum <= u * cum[:, -1:]).sum(-1)
    return torch.where(t[:, 0] > 0, token, index[:, 0])


# ── what a pass cannot do without ────────────────────────────────────────────

def _seq_tokens(case):
    """Expected tokens of all items of an attention case."""
    b, ctx = case["b"], case["ctx"]
    mean = (1 - 1 / 16) / math.log(16.0) if case["ragged"] else 1.0
    return ctx + (b - 1) * ctx * mean


def work(case):
    kind = case["kind"]
    if kind == "int4":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k // 2 + 2 * n * (k // case["gs"]) + 2 * m * k + 2 * m * n + (2 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    if kind == "append":
        n, hq, hkv, d, page = case["n"], case["hq"], case["hkv"], case["d"], case["page"]
        pages = -(-n // page) if case["prompt"] else n
        held = 2 * pages * page * hkv * d
        return {"bytes": 2 * n * (2 * hq + 2 * hkv) * d + 2 * n * hkv * (d + 2) + held * (1 + 2 / d) + 2 * held,
                "flops": 10 * n * (hq + hkv) * d}
    if kind == "attn":
        tok = _seq_tokens(case)
        return {"bytes": int(2 * tok * case["hkv"] * (case["d"] + 2)) + 4 * case["b"] * case["hq"] * case["d"],
                "flops": int(4 * tok * case["hq"] * case["d"])}
    return {"bytes": 2 * case["m"] * case["v"] + 12 * case["m"], "flops": 4 * case["m"] * case["v"]}


# ── the definitions in 64 bits ───────────────────────────────────────────────

def exact(case, seed):
    st = prepare(case, seed)
    return {"int4": _int4_exact, "append": _append_exact, "attn": _attn_exact, "sample": _sample_exact}[case["kind"]](st)


def _int4_exact(st):
    gs = st["case"]["gs"]
    x = st["x"].double()
    y = torch.zeros(x.shape[0], st["codes"].shape[0], dtype=torch.float64, device="cuda")
    for n0 in range(0, y.shape[1], 8192):            # (rows at a time: the doubles of a weight are large)
        w = st["codes"][n0:n0 + 8192].double() * st["scale"][n0:n0 + 8192].double().repeat_interleave(gs, 1)
        y[:, n0:n0 + 8192] = x @ w.t().contiguous()
    return y if st["bias"] is None else y + st["bias"].double()


def _append_exact(st):
    case = st["case"]
    n, hq, hkv, d, page = case["n"], case["hq"], case["hkv"], case["d"], case["page"]
    half = d // 2
    heads = st["qkv"].double().reshape(n, -1, d)
    turn = st["positions"].double().reshape(n, 1, 1) * st["inv_freq"].double()

    def rotated(x, w):
        x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / d + EPS) * w.double()
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * turn.cos() - b * turn.sin(), b * turn.cos() + a * turn.sin()], -1)

    def held(x):                                     # the values that codes and scale stand for
        s = (x.abs().max(-1, keepdim=True).values / 127).to(torch.float16).double()
        return torch.nan_to_num(torch.round(x / s).clamp(-127, 127) * s, nan=0.0)

    k_pool, v_pool, k_scale, v_scale = st["pool"]
    rows = st["slots"].long() * page + st["offsets"].long()
    out = []
    for codes, scale, new in ((k_pool, k_scale, rotated(heads[:, hq:hq + hkv], st["k_norm"])),
                              (v_pool, v_scale, heads[:, hq + hkv:])):
        old = (codes.double() * scale.double().unsqueeze(-1)).transpose(1, 2).reshape(-1, hkv, d)
        old[rows] = held(new)
        out.append(old.view(-1, page, hkv, d).transpose(1, 2)[st["pages"].long()])
    return rotated(heads[:, :hq], st["q_norm"]), out[0], out[1]


def _attn_exact(st):
    case = st["case"]
    b, hq, hkv, d, page = case["b"], case["hq"], case["hkv"], case["d"], case["page"]
    k_pool, v_pool, k_scale, v_scale = st["pool"]
    out = torch.zeros(b, hq, d, dtype=torch.float64, device="cuda")
    for i, n in enumerate(st["seq_lens"].tolist()):
        pages = st["page_table"][i, :-(-n // page)].long()
        for h in range(hkv):
            k = (k_pool[pages, h].double() * k_scale[pages, h].double().unsqueeze(-1)).reshape(-1, d)[:n]
            v = (v_pool[pages, h].double() * v_scale[pages, h].double().unsqueeze(-1)).reshape(-1, d)[:n]
            group = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            score = st["q"][i, group].double() @ k.t().contiguous() / d ** 0.5
            out[i, group] = torch.softmax(score, -1) @ v
    return out


def _sample_exact(st):
    logits = st["logits"].double().cpu().numpy()
    m, v = logits.shape
    u = st["u"].cpu().numpy()

    def rows(x, dtype):
        return x.cpu().numpy().astype(dtype) if torch.is_tensor(x) else np.full(m, x, dtype)
    ts, ks = rows(st["temperature"], np.float32), rows(st["top_k"], np.int64)
    ps, lows = rows(st["top_p"], np.float32), rows(st["min_p"], np.float32)
    tokens = []
    for i in range(m):
        row = logits[i]
        if ts[i] <= 0:
            tokens.append(int(np.flatnonzero(row == row.max())[0]))
            continue
        w = np.exp((row - row.max()).astype(np.longdouble) / np.longdouble(ts[i]))
        order = np.lexsort((np.arange(v), -row))
        if ks[i] > 0:
            order = order[:ks[i]]
        if ps[i] < 1:                                # the shortest prefix that holds a share p of the mass
            mass = np.cumsum(w[order])
            order = order[:max(1, 1 + int(np.count_nonzero(mass[:-1] < np.longdouble(ps[i]) * mass[-1])))]
        order = np.sort(order[(w[order] >= np.longdouble(lows[i])) | (order == order[0])])
        mass = np.cumsum(w[order])
        tokens.append(int(order[np.searchsorted(mass, np.longdouble(u[i]) * mass[-1], side="right")]))
    return torch.tensor(tokens)
