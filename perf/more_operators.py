"""Performance cases of the operators that serve chunks of new tokens over shared pages.

  chunk    attention of a ragged batch of new tokens, from a few drafted tokens to whole
           prompts and both in one batch, over a paged cache; with a sliding window and a
           few first tokens that stay visible where a model has them
  decode   the same for one new token of each sequence
  rope     rotary positions (half and interleaved layouts, part of the head, scaled
           frequencies), the norms of q and k where a model has them, and the new K/V into
           the pages of a ragged batch
  copy     pages copied inside a pool, as compaction moves them
  fork     sequences that continue others: page-table rows, and a page of their own for
           the tokens to come

The plain forms are elementary torch operations in fp32 (fp64 for the angles of far
positions).  `exact` is each operator's definition in fp64.
"""
import math
import random

import numpy as np
import torch

own = False

# q heads, kv heads, head dim
HEADS = [(32, 8, 128), (40, 8, 128), (64, 8, 128), (16, 8, 64), (32, 32, 64), (16, 1, 128)]
EPS = 1e-6


def listed():
    big = {"hq": 32, "hkv": 8, "d": 128, "page": 16}
    wide = {"hq": 40, "hkv": 8, "d": 128, "page": 16}
    return [
        # drafted tokens of a few sequences to verify: latency counts
        {"name": "chunk_drafts", "kind": "chunk", "b": 4, "new": 5, "ctx": 1500, "mix": "same", "window": 0,
         "sinks": 0, "pad": 0, **big},
        # a continuous batch: one prompt's chunk among decoding sequences, rows padded for a captured graph
        {"name": "chunk_mixed", "kind": "chunk", "b": 25, "new": 700, "ctx": 8000, "mix": "mixed", "window": 0,
         "sinks": 0, "pad": 44, **wide},
        # prompts of different lengths under a window, odd sizes
        {"name": "chunk_window", "kind": "chunk", "b": 3, "new": 7001, "ctx": 515, "mix": "ragged", "window": 1024,
         "sinks": 4, "pad": 0, **big},
        # a long prompt's last chunk: the largest case
        {"name": "chunk_long", "kind": "chunk", "b": 1, "new": 4096, "ctx": 12288, "mix": "same", "window": 0,
         "sinks": 0, "pad": 0, **wide},
        # single-stream decode far into a context, pages behind the window freed
        {"name": "decode_1", "kind": "decode", "b": 1, "ctx": 16384, "mix": "same", "window": 4096, "sinks": 4, **big},
        # a serving batch of different lengths, most of them past the window
        {"name": "decode_batch", "kind": "decode", "b": 16, "ctx": 12000, "mix": "ragged", "window": 2048,
         "sinks": 16, **wide},
        # one new token of each sequence; a quarter of the head turns, interleaved pairs
        {"name": "rope_decode", "kind": "rope", "b": 16, "new": 1, "ctx": 90000, "mix": "ragged", "rot": 32,
         "inter": True, "scaled": False, "norm": False, **big},
        # prompts with norms and frequencies scaled for a long context
        {"name": "rope_prompts", "kind": "rope", "b": 4, "new": 2000, "ctx": 1003, "mix": "ragged", "rot": 128,
         "inter": False, "scaled": True, "norm": True, **wide},
        # a few pages that a step's bookkeeping moves
        {"name": "copy_few", "kind": "copy", "n": 5, "hkv": 8, "d": 128, "page": 16},
        # compaction of a pool
        {"name": "copy_many", "kind": "copy", "n": 2048, "hkv": 8, "d": 128, "page": 16},
        # four beams of one layer's table
        {"name": "fork_beams", "kind": "fork", "rows": 4, "group": 4, "ctx": 1200, "hkv": 8, "d": 128, "page": 16},
        # sixteen beams over all layers' tables at once
        {"name": "fork_layers", "kind": "fork", "rows": 576, "group": 16, "ctx": 9000, "hkv": 8, "d": 128,
         "page": 16},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["chunk", "chunk", "decode", "rope", "copy", "fork"])
    hq, hkv, d = rng.choice(HEADS)
    page = rng.choice([16, 16, 32, 64])
    if kind in ("chunk", "decode"):
        windowed = kind == "decode" or rng.random() < 0.5
        case = {"kind": kind, "window": _log_int(rng, 1, 8192) if windowed else 0, "hq": hq, "hkv": hkv, "d": d,
                "page": page}
        case["sinks"] = rng.choice([0, 1, 4, 16, 100]) if windowed else 0
        if kind == "decode":
            case["b"] = _log_int(rng, 1, 32)
            case["ctx"] = _log_int(rng, 1, min(32768, 16 * 12000 * 8 // (case["b"] * hkv)))
            case["mix"] = rng.choice(["same", "ragged"])
            return case
        case["mix"] = rng.choice(["same", "ragged", "mixed"])
        case["b"] = _log_int(rng, 1, 32)
        cost = 4096 * 14336 * 40 * 128 / (hq * d)        # of the largest listed case, in (token, key) pairs
        case["new"] = _log_int(rng, 1, 4096 // (case["b"] if case["mix"] == "same" else 1))
        while True:
            case["ctx"] = _log_int(rng, 1, 16384) - 1
            if sum(n * (c + n / 2) for c, n in _sequences(case)) <= cost and \
                    sum(c + n for c, n in _sequences(case)) * hkv <= 16 * 12000 * 8:
                break
            case["new"] = max(1, case["new"] // 2)
        case["pad"] = rng.choice([0, 0, rng.randrange(1, 64)])
        return case
    if kind == "rope":
        b = _log_int(rng, 1, 32)
        decode = rng.random() < 0.4
        return {"kind": kind, "b": b, "new": 1 if decode else _log_int(rng, 1, max(1, 4000 // b)),
                "ctx": _log_int(rng, 1, 120000) - 1, "mix": rng.choice(["same", "ragged", "mixed"]),
                "rot": rng.choice([d, d, d // 2, d // 4, 2 * rng.randrange(1, d // 2 + 1)]),
                "inter": rng.random() < 0.5, "scaled": rng.random() < 0.5, "norm": rng.random() < 0.4,
                "hq": hq, "hkv": hkv, "d": d, "page": page}
    if kind == "copy":
        n = _log_int(rng, 1, max(1, 2048 * 8 * 128 * 16 // (hkv * d * page)))
        return {"kind": kind, "n": n, "hkv": hkv, "d": d, "page": page}
    group = rng.randrange(1, 17)
    groups = _log_int(rng, 1, max(1, 576 * 8 * 128 * 16 // (hkv * d * page * group)))
    return {"kind": kind, "rows": group * groups, "group": group, "ctx": _log_int(rng, 1, 9000), "hkv": hkv, "d": d,
            "page": page}


# ── what a case is made of ───────────────────────────────────────────────────

def _sequences(case):
    """(cached tokens, new tokens) of each sequence: all alike, or spread down to a
    sixteenth; "mixed": a chunk of the first one, one token of each of the others."""
    b, new, ctx, mix = case["b"], case.get("new", 1), case["ctx"], case["mix"]
    r = random.Random(f"{b} {new} {ctx} {mix}")
    out = [(ctx, new)]
    for _ in range(b - 1):
        c, n = int(ctx * 16.0 ** -r.random()), max(1, int(new * 16.0 ** -r.random()))
        out.append((ctx, new) if mix == "same" else (c, 1 if mix == "mixed" else n))
    return out


def _visible(case, pos):
    """Keys that the token at `pos` sees."""
    w, s = case["window"], case["sinks"]
    return pos + 1 if not w else min(pos + 1, w) + min(max(pos + 1 - w, 0), s)


def _pairs(case):
    """(new token, visible key) pairs of a case, and the tokens of its caches that any of them sees."""
    pairs = keys = 0
    for c, n in _sequences(case):
        pairs += sum(_visible(case, p) for p in range(c, c + n))
        keys += min(c + n, _visible(case, c) + n - 1) if case["window"] else c + n
    return pairs, keys


def _fork_rows(case):
    """Length of each row, its parent, and whether the child gets a page of its own
    (the first child of a parent goes on in the parent's)."""
    rows, group = case["rows"], case["group"]
    r = random.Random(f"{rows} {group} {case['ctx']}")
    lens = [max(1, int(case["ctx"] * 16.0 ** -r.random())) for _ in range(rows)]
    parents = [i // group * group + r.randrange(group) for i in range(rows)]
    seen, own_page = set(), []
    for p in parents:
        own_page.append(p in seen)
        seen.add(p)
    return lens, parents, own_page


# ── inputs ───────────────────────────────────────────────────────────────────

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).half()


def _pool(g, slots, hkv, page, d):
    """K and V pages [slots, Hkv, P, D] of about N(0, 1) (V stored with the tokens of a dim adjacent)."""
    return _normal(g, slots, hkv, page, d), _normal(g, slots, hkv, d, page).transpose(-1, -2)


def _ints(values):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(values, dtype=np.int32))).cuda()


def _tables(case, g, keep):
    """Page table [B, columns] of shuffled slots for the pages that keep(cached, new)
    names, -1 elsewhere (columns past the longest sequence, as tables have), and the
    number of slots."""
    page, seqs = case["page"], _sequences(case)
    table = np.full((len(seqs), max(-(-(c + n) // page) for c, n in seqs) + 3), -1, np.int64)
    used = 0
    for i, (c, n) in enumerate(seqs):
        j = np.arange(-(-(c + n) // page))
        j = j[keep(c, n, j)]
        table[i, j] = used + np.arange(len(j))
        used += len(j)
    order = torch.randperm(used + 5, generator=g, device="cuda").int()     # (a few slots of other sequences)
    t = torch.from_numpy(table).cuda()
    return torch.where(t >= 0, order[t.clamp(min=0)], torch.full_like(t, -1).int()).int().contiguous(), used + 5


def _scaled_inv_freq(rot, theta, factor, first_context):
    """Frequencies for a context `factor` times the first one: those that turn often in
    the first context stay, those that never complete a turn are divided by the factor,
    a ramp between (1 to 32 turns); and the factor that q and k are multiplied by."""
    inv = 1.0 / theta ** (np.arange(0, rot, 2) / rot)
    turns = first_context * inv / (2 * math.pi)
    stay = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
    return inv * stay + inv / factor * (1 - stay), 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    st = {"case": case}
    hkv, d, page = case["hkv"], case["d"], case["page"]
    if kind in ("chunk", "decode", "rope"):
        seqs = _sequences(case)
        n = sum(s[1] for s in seqs)
        st["seqs"] = seqs
        st["seq_lens"] = _ints([c + k for c, k in seqs])
        st["q_starts"] = _ints(np.concatenate([[0], np.cumsum([k for _, k in seqs])]))
    if kind in ("chunk", "decode"):
        w, s = case["window"], case["sinks"]

        def keep(c, k, j):                              # what has left every window is freed
            return (j * page < s) | ((j + 1) * page > (c - w + 1 if w else 0))
        st["page_table"], slots = _tables(case, g, keep)
        rows = n + case.get("pad", 0)
        st["q"] = _normal(g, rows, case["hq"], d)
        st["pool"] = _pool(g, slots, hkv, page, d)
        st["out"] = torch.zeros(rows, case["hq"], d, dtype=torch.float16, device="cuda")
        st["max_new"] = max(k for _, k in seqs)
    elif kind == "rope":
        st["page_table"], slots = _tables(case, g, lambda c, k, j: j >= c // page)
        st["pool"] = _pool(g, slots, hkv, page, d)
        st["qkv"] = _normal(g, n, (case["hq"] + 2 * hkv) * d)
        st["norms"] = [(1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")).half() if case["norm"] else None
                       for _ in range(2)]
        inv, st["rope_scale"] = (_scaled_inv_freq(case["rot"], 1e6, 4.0, 32768) if case["scaled"]
                                 else (1.0 / 1e4 ** (np.arange(0, case["rot"], 2) / case["rot"]), 1.0))
        st["inv_freq"] = torch.from_numpy(inv.astype(np.float32)).cuda()
        st["q_out"] = torch.empty(n, case["hq"], d, dtype=torch.float16, device="cuda")
    elif kind == "copy":
        n = case["n"]
        slots = 2 * n + max(1, n // 8)
        order = torch.randperm(slots, generator=g, device="cuda").int()
        st["src"], st["dst"] = order[:n].contiguous(), order[n:2 * n].contiguous()
        st["pool"] = _pool(g, slots, hkv, page, d)
    else:
        # rows of a group share their full pages (as beams do): a prefix of one list, then their own last page
        lens, parents, own_page = _fork_rows(case)
        cols = case["ctx"] // page + 2
        table = np.full((case["rows"], cols), -1, np.int32)
        r = random.Random(int(seed))
        shared = 64
        for i, length in enumerate(lens):
            table[i, :length // page] = np.random.default_rng(seed * 1009 + i).integers(0, shared, length // page)
            table[i, length // page] = shared + i
        fresh = [shared + case["rows"] + i if o else -1 for i, o in enumerate(own_page)]
        slots = shared + 2 * case["rows"]
        order = list(range(slots))
        r.shuffle(order)
        order = np.asarray(order + [-1], np.int32)      # (entry -1 stays -1)
        st["page_table"], st["seq_lens"] = _ints(order[table]), _ints(lens)
        st["parents"], st["fresh"] = _ints(parents), _ints(order[fresh])
        st["pool"] = _pool(g, slots, hkv, page, d)
        st["table_out"], st["lens_out"] = torch.empty_like(st["page_table"]), torch.empty_like(st["seq_lens"])
    if own:       # the view of its pool and the workspace that a program keeps
        from helm_amd.kernels import attention as ka
        st["view"] = ka.PoolView.of_pool(*st["pool"])
        st["workspace"] = ka.AttnWorkspace(st["pool"][0].device)
    return st


# ── one pass ─────────────────────────────────────────────────────────────────

def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    from helm_amd.kernels import attention as ka
    from helm_amd.kernels import fused

    case, kind = st["case"], st["case"]["kind"]
    if kind == "chunk":
        return ka.chunk_attention(st["q"], st["view"], st["page_table"], st["seq_lens"], st["q_starts"], case["page"],
                                  window=case["window"], sinks=case["sinks"], max_new=st["max_new"],
                                  workspace=st["workspace"], out=st["out"])
    if kind == "decode":
        return ka.window_decode_attention(st["q"], st["view"], st["page_table"], st["seq_lens"], case["page"],
                                          case["window"], case["sinks"], workspace=st["workspace"], out=st["out"])
    if kind == "rope":
        q = fused.rope_append(st["qkv"], st["view"], st["page_table"], st["seq_lens"], st["q_starts"], case["page"],
                              st["inv_freq"], case["hq"], case["hkv"], case["d"], interleaved=case["inter"],
                              rope_scale=st["rope_scale"], q_norm_w=st["norms"][0], k_norm_w=st["norms"][1], eps=EPS,
                              q_out=st["q_out"])
        return q, st["pool"][0], st["pool"][1]
    if kind == "copy":
        ka.copy_pages(st["view"], st["src"], st["dst"], case["page"])
        return st["pool"]
    table, lens = ka.fork_pages(st["view"], st["page_table"], st["seq_lens"], st["parents"], st["fresh"], case["page"],
                                table_out=st["table_out"], lens_out=st["lens_out"])
    return table, lens, st["pool"][0], st["pool"][1]


def _run_plain(st):
    return {"chunk": _attend, "decode": _attend, "rope": _rope, "copy": _copy, "fork": _fork}[st["case"]["kind"]](st)


def _attend(st):
    case = st["case"]
    hq, hkv, d, page, w, s = (case[x] for x in ("hq", "hkv", "d", "page", "window", "sinks"))
    k_pool, v_pool = st["pool"]
    out, row = st["out"], 0
    inside = torch.arange(page, device="cuda")
    for i, (c, n) in enumerate(st["seqs"]):
        pages = -(-(c + n) // page)
        # the pages that any of its tokens sees
        j = torch.arange(pages, device="cuda")
        if w:
            lo = max(0, c - w + 1) // page
            first = min(lo, -(-s // page))
            j = torch.cat([j[:first], j[lo:]])
        slots = st["page_table"][i][j].long()
        key = (j[:, None] * page + inside).reshape(-1)
        k = k_pool[slots].permute(1, 0, 2, 3).reshape(hkv, -1, d).float()
        v = v_pool[slots].permute(1, 0, 2, 3).reshape(hkv, -1, d).float()
        v = torch.where((key < c + n)[:, None], v, torch.zeros_like(v))
        kt = k.transpose(1, 2).contiguous()
        for t in range(0, n, 512):
            m = min(512, n - t)
            q = st["q"][row + t:row + t + m].float().view(m, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
            pos = torch.arange(c + t, c + t + m, device="cuda")[:, None]
            seen = key <= pos
            if w:
                seen &= (key > pos - w) | (key < s)
            score = (torch.matmul(q, kt) / math.sqrt(d)).view(hkv, -1, m, len(key))
            score = score.masked_fill(~seen, -math.inf)
            p = torch.exp(score - score.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            o = torch.matmul(p.view(hkv, -1, len(key)), v).view(hkv, -1, m, d)
            out[row + t:row + t + m] = o.permute(2, 0, 1, 3).reshape(m, hq, d).half()
        row += n
    return out


def _places(st):
    """Row, position, slot and offset of each new token."""
    page = st["case"]["page"]
    starts, lens = st["q_starts"].long(), st["seq_lens"].long()
    row = torch.arange(st["qkv"].shape[0], device="cuda")
    seq = (row[:, None] >= starts[1:]).sum(-1)
    pos = lens[seq] - starts[seq + 1] + row
    return pos, st["page_table"][seq, pos // page].long(), pos % page


def _rope(st):
    case = st["case"]
    hq, hkv, d, rot = case["hq"], case["hkv"], case["d"], case["rot"]
    x = st["qkv"].float().view(-1, hq + 2 * hkv, d)
    qk, v = x[:, :hq + hkv], x[:, hq + hkv:]
    if case["norm"]:
        wt = torch.cat([st["norms"][0].float().expand(hq, d), st["norms"][1].float().expand(hkv, d)])
        qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS) * wt
    pos, slots, offs = _places(st)
    ang = pos.double()[:, None] * st["inv_freq"].double()
    c, s = ((f(ang) * st["rope_scale"]).float()[:, None] for f in (torch.cos, torch.sin))
    turn, rest = qk[..., :rot], qk[..., rot:]
    if case["inter"]:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = turn[..., :rot // 2], turn[..., rot // 2:]
        turn = torch.cat([a * c - b * s, b * c + a * s], -1)
    qk = torch.cat([turn, rest], -1).half()
    k_pool, v_pool = st["pool"]
    k_pool[slots, :, offs] = qk[:, hq:]
    v_pool[slots, :, offs] = v.half()
    return qk[:, :hq], k_pool, v_pool


def _copy(st):
    src, dst = st["src"].long(), st["dst"].long()
    for x in st["pool"]:
        x[dst] = x[src]
    return st["pool"]


def _fork(st):
    case = st["case"]
    page = case["page"]
    parents, fresh = st["parents"].long(), st["fresh"].long()
    rows, lens = st["page_table"][parents], st["seq_lens"][parents]
    col = torch.arange(rows.shape[1], device="cuda")
    tail = (lens // page).long()[:, None]
    own_page = (fresh >= 0)[:, None]
    table = torch.where(own_page & (col > tail), torch.full_like(rows, -1), rows)
    table = torch.where(own_page & (col == tail), fresh[:, None].int(), table)
    src = rows.gather(1, tail)[:, 0].long()
    put = (fresh >= 0) & (lens % page != 0)
    src, dst = src[put], fresh[put]
    for x in st["pool"]:
        x[dst] = x[src]
    return table, lens, st["pool"][0], st["pool"][1]


# ── what a pass cannot do without ────────────────────────────────────────────

def work(case):
    kind, hkv, d, page = case["kind"], case["hkv"], case["d"], case["page"]
    held = 4 * hkv * page * d                            # bytes of a page's K and V
    if kind in ("chunk", "decode"):
        pairs, keys = _pairs(case)
        new = sum(n for _, n in _sequences(case))
        return {"bytes": 4 * keys * hkv * d + 4 * new * case["hq"] * d, "flops": 4 * pairs * case["hq"] * d}
    if kind == "rope":
        n = sum(k for _, k in _sequences(case))
        return {"bytes": 4 * n * (case["hq"] + 2 * hkv) * d, "flops": 6 * n * (case["hq"] + hkv) * d}
    if kind == "copy":
        return {"bytes": 2 * case["n"] * held + 8 * case["n"], "flops": 0}
    lens, parents, own_page = _fork_rows(case)
    copies = sum(1 for p, o in zip(parents, own_page) if o and lens[p] % page)
    return {"bytes": 2 * copies * held + sum(8 * (lens[p] // page + 1) for p in parents) + 16 * len(lens), "flops": 0}


# ── the definitions in 64 bits ───────────────────────────────────────────────

def exact(case, seed):
    st = prepare(case, seed)
    return {"chunk": _attend_exact, "decode": _attend_exact, "rope": _rope_exact, "copy": _copy_exact,
            "fork": _fork_exact}[case["kind"]](st)


def _attend_exact(st):
    case = st["case"]
    group, d, page = case["hq"] // case["hkv"], case["d"], case["page"]
    out = st["out"].double()
    starts = st["q_starts"].tolist()
    for i, length in enumerate(st["seq_lens"].tolist()):
        n = starts[i + 1] - starts[i]
        for t0 in range(0, n, 256):
            rows = range(t0, min(n, t0 + 256))
            first, last = length - n + rows[0], length - n + rows[-1]
            lo = max(0, first - case["window"] + 1) if case["window"] else 0
            keys = list(range(min(case["sinks"], lo))) + list(range(lo, last + 1))
            key = torch.tensor(keys, device="cuda")
            slot = st["page_table"][i, key // page].long()
            pos = torch.arange(first, last + 1, device="cuda").view(-1, 1)
            hidden = key > pos
            if case["window"]:
                hidden = hidden | ((pos - key >= case["window"]) & (key >= case["sinks"]))
            q0 = starts[i] + rows[0]
            for h in range(case["hkv"]):
                k = st["pool"][0][slot, h, key % page].double()
                v = st["pool"][1][slot, h, key % page].double()
                for hh in range(h * group, (h + 1) * group):
                    x = st["q"][q0:q0 + len(rows), hh].double() @ k.t().contiguous() / d ** 0.5
                    x[hidden] = -math.inf
                    out[q0:q0 + len(rows), hh] = torch.softmax(x, -1) @ v
    return out


def _rope_exact(st):
    case = st["case"]
    hq, hkv, d, page, rot = (case[x] for x in ("hq", "hkv", "d", "page", "rot"))
    heads = st["qkv"].double().reshape(-1, hq + 2 * hkv, d)
    pos, slot = [], []
    table = st["page_table"].cpu().numpy()
    for i, (c, n) in enumerate(_sequences(case)):
        p = np.arange(c, c + n)
        pos.append(p)
        slot.append(table[i, p // page])
    pos, slot = np.concatenate(pos), torch.from_numpy(np.concatenate(slot)).cuda().long()
    turn = torch.from_numpy(pos.astype(np.float64)).cuda().view(-1, 1) * st["inv_freq"].double()
    unit = torch.polar(torch.full_like(turn, st["rope_scale"]), turn).unsqueeze(1)

    def rotated(x, w):
        x = x.clone()
        if w is not None:
            x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / d + EPS) * w.double()
        at = torch.arange(rot, device="cuda")
        re, im = (at[0::2], at[1::2]) if case["inter"] else (at[:rot // 2], at[rot // 2:])
        z = torch.complex(x[..., re], x[..., im]) * unit
        x[..., re], x[..., im] = z.real, z.imag
        return x
    rows = slot * page + torch.from_numpy(pos % page).cuda()
    out = [rotated(heads[:, :hq], st["norms"][0])]
    for held, new in ((st["pool"][0], rotated(heads[:, hq:hq + hkv], st["norms"][1])),
                      (st["pool"][1], heads[:, hq + hkv:])):
        flat = held.double().transpose(1, 2).reshape(-1, hkv, d)
        flat[rows] = new
        out.append(flat.view(-1, page, hkv, d).transpose(1, 2))
    return tuple(out)


def _moved(pool, src, dst):
    at = torch.arange(pool[0].shape[0], device="cuda")
    at[torch.tensor(dst, device="cuda", dtype=torch.long)] = torch.tensor(src, device="cuda", dtype=torch.long)
    return tuple(x.double()[at] for x in pool)


def _copy_exact(st):
    return _moved(st["pool"], st["src"].tolist(), st["dst"].tolist())


def _fork_exact(st):
    page = st["case"]["page"]
    table, lens = st["page_table"].cpu().numpy(), st["seq_lens"].tolist()
    rows, out_lens, src, dst = [], [], [], []
    for p, f in zip(st["parents"].tolist(), st["fresh"].tolist()):
        row, full = table[p].copy(), lens[p] // page
        if f >= 0:
            if lens[p] % page:
                src.append(int(row[full]))
                dst.append(f)
            row[full] = f
            row[full + 1:] = -1
        rows.append(row)
        out_lens.append(lens[p])
    return (_ints(np.stack(rows)), _ints(out_lens)) + _moved(st["pool"], src, dst)
