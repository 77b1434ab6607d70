"""Cases of the tree-verification operators, each with a plain torch form.

A draft model proposes a tree of tokens for every request of a decode step. The target model writes their cache
rows behind the request's context, rotates their queries to the positions of their depths, attends every draft to
the context and to its own ancestors (``tree_mla_decode``), and moves the rows of the accepted path together
(``commit_draft_rows``). Chunked prefill and cache transfer read the quantised rows back (``gather_cache``).
"""
import math

import torch

own = False

PAGE = 64
LATENT, ROPE = 512, 64
WIDTH = LATENT + ROPE
ROW_BYTES = {"ds_mla": 656, "idxk": 132, "bf16": 1152, "f16": 1152}
ROW_VALUES = {"ds_mla": 576, "idxk": 128, "bf16": 576, "f16": 576}
DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SCALE = 192 ** -0.5  # softmax scale of the attention this repository serves (128 + 64 dims a head)


def listed():
    return [
        # a request's first drafts behind a short prompt: latency
        {"name": "tree_short", "op": "tree", "batch": 1, "drafts": 4, "heads": 8, "context": 37, "cache": "ds_mla",
         "dtype": "bf16", "ragged": False},
        # a decode step of a rank that holds 8 of 64 heads, requests of different ages and tree sizes
        {"name": "tree_heads8_ragged", "op": "tree", "batch": 8, "drafts": 16, "heads": 8, "context": 24576,
         "cache": "ds_mla", "dtype": "bf16", "ragged": True},
        # all heads on one GPU, small trees
        {"name": "tree_heads64", "op": "tree", "batch": 4, "drafts": 8, "heads": 64, "context": 24576,
         "cache": "ds_mla", "dtype": "f16", "ragged": False},
        # one long context, a wide tree
        {"name": "tree_long", "op": "tree", "batch": 1, "drafts": 32, "heads": 64, "context": 131072,
         "cache": "ds_mla", "dtype": "bf16", "ragged": False},
        # an unquantised cache, odd sizes
        {"name": "tree_bf16_cache", "op": "tree", "batch": 5, "drafts": 7, "heads": 16, "context": 8191,
         "cache": "bf16", "dtype": "bf16", "ragged": True},
        # rotary part of a decode step's queries, into the attention's query rows
        {"name": "rope_decode", "op": "rope", "tokens": 16, "heads": 64, "width": 64, "rotary": 64, "offset": 0,
         "row_in": 256, "row_out": 576, "neox": False, "dtype": "bf16", "positions": 180224, "factor": 40.0},
        # the same of a prefill
        {"name": "rope_prefill", "op": "rope", "tokens": 16384, "heads": 64, "width": 64, "rotary": 64, "offset": 0,
         "row_in": 256, "row_out": 576, "neox": False, "dtype": "bf16", "positions": 180224, "factor": 40.0},
        # whole heads with a rotary first half (the indexer's queries), half layout
        {"name": "rope_half_heads", "op": "rope", "tokens": 4097, "heads": 32, "width": 128, "rotary": 64, "offset": 0,
         "row_in": 128, "row_out": 128, "neox": True, "dtype": "f16", "positions": 131072, "factor": 1.0},
        # a long context read back for a prefill chunk
        {"name": "gather_latent", "op": "gather", "batch": 1, "context": 131072, "cache": "ds_mla", "dtype": "bf16",
         "ragged": False},
        # indexer keys of a ragged batch
        {"name": "gather_indexer", "op": "gather", "batch": 7, "context": 4099, "cache": "idxk", "dtype": "f16",
         "ragged": True},
        # accepted paths of a batch, the caches of many layers
        {"name": "commit_layers", "op": "commit", "batch": 8, "drafts": 32, "layers": 48, "cache": "ds_mla"},
        # one request, one layer
        {"name": "commit_one", "op": "commit", "batch": 1, "drafts": 4, "layers": 1, "cache": "idxk"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "rope", "gather", "commit"])
    if op == "tree":
        drafts, heads = _log(rng, 1, 64), rng.choice([4, 8, 13, 16, 32, 64, 128])
        batch = _log(rng, 1, 24)
        most = min(131072, 196608 // batch, 2048 * 131072 // (batch * drafts * heads))
        context = _log(rng, 1, max(1, most - drafts)) + drafts
        cache = rng.choice(["ds_mla", "ds_mla", "bf16", "f16"])
        dtype = cache if cache in DTYPE else rng.choice(["bf16", "f16"])
        return {"op": op, "batch": batch, "drafts": drafts, "heads": heads, "context": context, "cache": cache,
                "dtype": dtype, "ragged": rng.random() < 0.5}
    if op == "rope":
        rotary = rng.choice([32, 64, 96, 128])
        offset = rng.choice([0, 0, 16, 64])
        width = offset + rotary + rng.choice([0, 8, 64])
        heads = rng.choice([1, 2, 7, 16, 64])
        return {"op": op, "tokens": _log(rng, 1, max(1, 2 ** 26 // (heads * width))), "heads": heads, "width": width,
                "rotary": rotary, "offset": offset, "row_in": width + rng.choice([0, 64, 192]),
                "row_out": width + rng.choice([0, 8, 512]), "neox": rng.random() < 0.5,
                "dtype": rng.choice(["bf16", "f16", "f32"]), "positions": _log(rng, 64, 180224),
                "factor": rng.choice([1.0, 4.0, 40.0])}
    if op == "gather":
        batch = _log(rng, 1, 32)
        cache = rng.choice(["ds_mla", "idxk", "bf16", "f16"])
        return {"op": op, "batch": batch, "context": _log(rng, 1, 131072 // batch), "cache": cache,
                "dtype": cache if cache in ("bf16", "f16") else rng.choice(["bf16", "f16"]),
                "ragged": rng.random() < 0.5}
    return {"op": op, "batch": _log(rng, 1, 32), "drafts": _log(rng, 1, 64), "layers": _log(rng, 1, 48),
            "cache": rng.choice(["ds_mla", "idxk", "bf16"])}


def _lengths(case):
    """Positions of each request, drafts among them, and its drafts."""
    n, context, drafts = case["batch"], case["context"], case.get("drafts", 1)
    if not case["ragged"]:
        return [context] * n, [drafts] * n
    lens = [max(min(drafts, context), context - (context * b) // (2 * n)) for b in range(n)]
    return lens, [max(1, drafts - (drafts * b) // (2 * n)) for b in range(n)]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _quantised(rows, g, values):
    """`rows` cache rows of N(0, 1) values: e4m3 codes and f32 scales (amax / 448 of each 128 values), then the
    latent row's 64 rotary values in half."""
    out = torch.empty(rows, 656 if values == WIDTH else 132, dtype=torch.uint8, device="cuda")
    groups = (4 if values == WIDTH else 1)
    for lo in range(0, rows, 65536):
        hi = min(rows, lo + 65536)
        x = torch.randn(hi - lo, groups, 128, generator=g, device="cuda")
        s = x.abs().amax(dim=2, keepdim=True) / 448.0
        out[lo:hi, :128 * groups] = (x / s).to(torch.float8_e4m3fn).view(torch.uint8).reshape(hi - lo, -1)
        out[lo:hi, 128 * groups:132 * groups] = s.reshape(hi - lo, groups).contiguous().view(torch.uint8)
        if values == WIDTH:
            pe = torch.randn(hi - lo, ROPE, generator=g, device="cuda").half()
            out[lo:hi, 528:] = pe.view(torch.uint8)
    return out


def _pool(case, g, pages):
    values = ROW_VALUES[case["cache"]]
    if case["cache"] in ("ds_mla", "idxk"):
        return _quantised(pages * PAGE, g, values).view(pages, PAGE, -1)
    return torch.randn(pages, PAGE, values, generator=g, device="cuda", dtype=DTYPE[case["cache"]])


def _tables(lens, g, spare=1):
    """A block table of randomly placed pages, and how many pages the pool needs."""
    need = [-(-n // PAGE) for n in lens]
    width, total = max(need) + spare, sum(need) + 3
    order = torch.randperm(total, generator=g, device="cuda").int()
    at = torch.arange(width, device="cuda")
    first = torch.tensor([sum(need[:b]) for b in range(len(need))], device="cuda")
    used = at[None, :] < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(used, order[(first[:, None] + at[None, :]).clamp(max=total - 1)], torch.zeros((), dtype=torch.int32, device="cuda"))
    return table.contiguous(), total


def _parents(n, drafts, g):
    """Random trees: draft i's parent is an earlier draft or, -1, the context's last token."""
    u = torch.rand(n, drafts, generator=g, device="cuda")
    return (u * (torch.arange(drafts, device="cuda") + 1)).floor().long().clamp(max=drafts - 1) - 1


def _ancestors(parents):
    """Bit j of [b, i]: draft j is i or an ancestor of i."""
    n, drafts = parents.shape
    bits = torch.ones((), dtype=torch.int64, device=parents.device) << torch.arange(drafts, device=parents.device)
    mask = bits.expand(n, drafts).clone()
    for i in range(1, drafts):
        p = parents[:, i]
        above = mask.gather(1, p.clamp(min=0)[:, None])[:, 0]
        mask[:, i] |= torch.where(p >= 0, above, torch.zeros_like(above))
    return mask


def _cos_sin(rotary, positions, factor):
    """cos | sin of every position, f32 of angles in 64 bits; factor > 1: frequencies interpolated by parts."""
    i = torch.arange(rotary // 2, device="cuda", dtype=torch.float64)
    freq = 10000.0 ** (-2.0 * i / rotary)
    gain = 1.0
    if factor > 1.0:
        turns = 4096.0 * freq / (2.0 * math.pi)  # over the original context
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        freq = freq * keep + freq / factor * (1.0 - keep)
        gain = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos() * gain, angle.sin() * gain], dim=1).float()


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    s = {"op": op, "case": case}
    if op == "tree":
        lens, drafts = _lengths(case)
        n, t, h = case["batch"], case["drafts"], case["heads"]
        s["table"], pages = _tables(lens, g)
        s["cache"] = _pool(case, g, pages)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["drafts"] = torch.tensor(drafts, dtype=torch.int32, device="cuda")
        s["q"] = torch.randn(n, t, h, WIDTH, generator=g, device="cuda").to(DTYPE[case["dtype"]])
        s["mask"] = _ancestors(_parents(n, t, g))
    elif op == "rope":
        dtype = DTYPE[case["dtype"]]
        t, h, lead_in, lead_out = case["tokens"], case["heads"], case["row_in"] - case["width"], case["row_out"] - case["width"]
        s["x"] = torch.randn(t, h, case["row_in"], generator=g, device="cuda").to(dtype)[:, :, lead_in:]
        s["out"] = torch.zeros(t, h, case["row_out"], device="cuda", dtype=dtype)[:, :, lead_out:]
        s["positions"] = torch.randint(0, case["positions"], (t,), generator=g, device="cuda")
        s["cos_sin"] = _cos_sin(case["rotary"], case["positions"], case["factor"])
    elif op == "gather":
        lens, _ = _lengths(case)
        s["table"], pages = _tables(lens, g)
        s["cache"] = _pool(case, g, pages)
        ends = torch.tensor([0] + lens, dtype=torch.int64).cumsum(0)
        s["starts"], s["total"] = ends.int().cuda(), int(ends[-1])
    else:
        n, t = case["batch"], case["drafts"]
        lens = [t + 100 + 7 * b for b in range(n)]
        s["table"], pages = _tables(lens, g)
        rows = case["layers"] * pages
        s["pool"] = _pool(case, g, rows).view(case["layers"], pages, PAGE, -1)
        s["caches"] = list(s["pool"].unbind(0))
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["drafts"] = torch.full((n,), t, dtype=torch.int32, device="cuda")
        # an accepted path: ascending drafts from the root down, -1 behind its end
        depth = max(1, (t + 1) // 2)
        took = torch.rand(n, t, generator=g, device="cuda").argsort(dim=1)[:, :depth].sort(dim=1).values
        length = torch.randint(1, depth + 1, (n, 1), generator=g, device="cuda")
        s["accepted"] = torch.where(torch.arange(depth, device="cuda")[None] < length, took, -1).int().contiguous()
    return s


# ---------------------------------------------------------------- plain forms
def _rows(table, positions):
    """Cache rows of positions [b, p] through the block table."""
    page = table.long().gather(1, (positions // PAGE).clamp(max=table.shape[1] - 1))
    return page * PAGE + positions % PAGE


def _dequantised(rows, cache):
    """Cache rows [..., row] as f32 values."""
    if cache in ("bf16", "f16"):
        return rows.float()
    groups = 4 if cache == "ds_mla" else 1
    lead = rows.shape[:-1]
    codes = rows[..., :128 * groups].contiguous().view(torch.float8_e4m3fn).float().view(*lead, groups, 128)
    scales = rows[..., 128 * groups:132 * groups].contiguous().view(torch.float32)
    values = (codes * scales[..., None]).flatten(-2)
    if cache == "idxk":
        return values
    return torch.cat([values, rows[..., 528:].contiguous().view(torch.float16).float()], dim=-1)


def _plain_tree(s):
    case = s["case"]
    n, t, h = case["batch"], case["drafts"], case["heads"]
    longest = case["context"]
    p = torch.arange(longest, device="cuda")[None].expand(n, -1)
    flat = s["cache"].view(-1, s["cache"].shape[-1])
    inside = p < s["lens"][:, None]
    kv = _dequantised(flat[_rows(s["table"], torch.where(inside, p, 0))], case["cache"])  # [b, p, 576]
    j = p - (s["lens"] - s["drafts"])[:, None]  # draft of each position; negative: context
    bit = (s["mask"][:, :, None] >> j.clamp(0, 63)[:, None, :]) & 1
    sees = ((j < 0)[:, None, :] | (bit == 1)) & inside[:, None, :]
    sees &= (torch.arange(t, device="cuda")[None] < s["drafts"][:, None])[:, :, None]  # [b, i, p]
    z = torch.bmm(s["q"].float().view(n, t * h, WIDTH), kv.transpose(1, 2)).view(n, t, h, longest)
    z.mul_(SCALE).masked_fill_(~sees[:, :, None, :], -math.inf)
    top = z.amax(dim=3, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = z.sub_(top).exp_()
    total = e.sum(dim=3, keepdim=True)
    o = torch.bmm(e.view(n, t * h, longest), kv[:, :, :LATENT]).view(n, t, h, LATENT)
    o = torch.where(total > 0, o / total.clamp(min=1e-37), torch.zeros_like(o))
    lse = (top + total.log())[..., 0]
    return o.to(s["q"].dtype), lse


def _plain_rope(s):
    case = s["case"]
    r, lo, x = case["rotary"], case["offset"], s["x"].float()
    cos, sin = s["cos_sin"][s["positions"]][:, None, :].split(r // 2, dim=2)
    part = x[:, :, lo:lo + r]
    if case["neox"]:
        a, b = part[:, :, :r // 2], part[:, :, r // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=2)
    else:
        a, b = part[:, :, 0::2], part[:, :, 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=3).flatten(2)
    return torch.cat([x[:, :, :lo], turned, x[:, :, lo + r:]], dim=2).to(s["x"].dtype)


def _plain_gather(s):
    at = torch.arange(s["total"], device="cuda")
    b = torch.searchsorted(s["starts"][1:].long(), at, right=True)
    p = at - s["starts"].long()[b]
    rows = s["table"].long()[b, p // PAGE] * PAGE + p % PAGE
    values = _dequantised(s["cache"].view(-1, s["cache"].shape[-1])[rows], s["case"]["cache"])
    return values.to(DTYPE[s["case"]["dtype"]])


def _plain_commit(s):
    pool = s["pool"].view(s["pool"].shape[0], -1, s["pool"].shape[-1])
    base = (s["lens"] - s["drafts"]).long()[:, None]
    taken = s["accepted"].long()
    k = torch.arange(taken.shape[1], device="cuda")[None].expand_as(taken)
    moved = taken >= 0
    src, dst = _rows(s["table"], base + taken.clamp(min=0))[moved], _rows(s["table"], base + k)[moved]
    pool[:, dst] = pool[:, src]
    return s["pool"]


def run(s):
    op = s["op"]
    if own:
        import importlib
        dsa = importlib.import_module("glm5-on-v100_b200")
        if op == "tree":
            o, lse = dsa.mla_sparse.forward_mqa_tree(s["q"], s["cache"], s["table"], s["lens"], s["mask"], SCALE,
                                                     draft_lens=s["drafts"])
            return {"o": o, "lse": lse}
        if op == "rope":
            dsa.rotary_embedding(s["out"], s["x"], s["positions"], s["cos_sin"], s["case"]["neox"], s["case"]["offset"])
            return {"out": s["out"]}
        if op == "gather":
            out = torch.empty(s["total"], ROW_VALUES[s["case"]["cache"]], dtype=DTYPE[s["case"]["dtype"]], device="cuda")
            dsa.gather_cache(out, s["cache"], s["table"], s["starts"])
            return {"out": out}
        dsa.commit_draft_rows(s["caches"], s["table"], s["lens"], s["accepted"], s["drafts"])
        return {"pool": s["pool"]}
    if op == "tree":
        o, lse = _plain_tree(s)
        return {"o": o, "lse": lse}
    if op == "rope":
        return {"out": _plain_rope(s)}
    if op == "gather":
        return {"out": _plain_gather(s)}
    return {"pool": _plain_commit(s)}


def work(case):
    op = case["op"]
    if op == "tree":
        lens, drafts = _lengths(case)
        rows = case["batch"] * case["drafts"] * case["heads"]
        seen = sum(lens)
        pairs = sum(a * d * case["heads"] for a, d in zip(lens, drafts))
        return {"bytes": seen * ROW_BYTES[case["cache"]] + rows * (WIDTH * 2 + LATENT * 2 + 4) + 4 * seen // PAGE,
                "flops": 2 * pairs * (WIDTH + LATENT)}
    if op == "rope":
        item = 4 if case["dtype"] == "f32" else 2
        t = case["tokens"]
        return {"bytes": t * (2 * case["heads"] * case["width"] * item + 4 * case["rotary"] + 8),
                "flops": 3 * t * case["heads"] * case["rotary"]}
    if op == "gather":
        seen = sum(_lengths(case)[0])
        values = ROW_VALUES[case["cache"]]
        return {"bytes": seen * (ROW_BYTES[case["cache"]] + 2 * values) + 4 * seen // PAGE,
                "flops": seen * values if case["cache"] in ("ds_mla", "idxk") else 0}
    accepted = case["batch"] * (1 + max(1, (case["drafts"] + 1) // 2)) / 2  # paths of 1 to (drafts + 1) / 2
    return {"bytes": int(2 * accepted * case["layers"] * ROW_BYTES[case["cache"]] + 4 * accepted), "flops": 0}


# ------------------------------------------------------------------ 64 bits
def _e4m3_values():
    code = torch.arange(256, device="cuda")
    e, m = (code >> 3 & 15).double(), (code & 7).double()
    v = torch.where(e == 0, m / 512.0, (1.0 + m / 8.0) * torch.exp2(e - 7.0))
    return torch.where(code >= 128, -v, v)


def _exact_row(raw, cache):
    if cache in ("bf16", "f16"):
        return raw.double()
    look, groups = _e4m3_values(), (4 if cache == "ds_mla" else 1)
    parts = []
    for k in range(groups):
        scale = raw[:, 128 * groups + 4 * k:128 * groups + 4 * k + 4].contiguous().view(torch.float32).double()
        parts.append(look[raw[:, 128 * k:128 * k + 128].long()] * scale)
    if cache == "ds_mla":
        parts.append(raw[:, 528:656].contiguous().view(torch.float16).double())
    return torch.cat(parts, dim=1)


def _positions_of(s, b, n):
    page = s["table"][b, :-(-n // PAGE)].long()
    return (page[:, None] * PAGE + torch.arange(PAGE, device="cuda")[None]).reshape(-1)[:n]


def exact(case, seed):
    op = case["op"]
    if op == "commit":
        return None
    s = prepare(case, seed)
    if op == "rope":
        r, lo, out = case["rotary"], case["offset"], s["x"].double()
        angle = s["cos_sin"].double()[s["positions"]]
        for i in range(r // 2):
            u, v = (lo + i, lo + i + r // 2) if case["neox"] else (lo + 2 * i, lo + 2 * i + 1)
            c, d = angle[:, i, None], angle[:, r // 2 + i, None]
            a, b = s["x"][:, :, u].double(), s["x"][:, :, v].double()
            out[:, :, u], out[:, :, v] = a * c - b * d, b * c + a * d
        return {"out": out}
    flat = s["cache"].view(-1, s["cache"].shape[-1])
    lens, drafts = _lengths(case)
    if op == "gather":
        return {"out": torch.cat([_exact_row(flat[_positions_of(s, b, n)], case["cache"]) for b, n in enumerate(lens)])}
    h = case["heads"]
    o = torch.zeros(case["batch"], case["drafts"], h, LATENT, dtype=torch.float64, device="cuda")
    lse = torch.full((case["batch"], case["drafts"], h), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        kv = _exact_row(flat[_positions_of(s, b, n)], case["cache"])
        for i in range(drafts[b]):
            word = int(s["mask"][b, i])
            keep = torch.tensor([bool(word >> j & 1) for j in range(drafts[b])], device="cuda")
            hidden = torch.zeros(n, dtype=torch.bool, device="cuda")
            first = n - drafts[b]
            hidden[max(first, 0):] = ~keep[max(-first, 0):]
            z = s["q"][b, i].double() @ kv.t() * SCALE
            z[:, hidden] = -math.inf
            lse[b, i] = torch.logsumexp(z, dim=1)
            o[b, i] = torch.exp(z - torch.where(lse[b, i].isinf(), torch.zeros_like(lse[b, i]), lse[b, i])[:, None]) @ kv[:, :LATENT]
    return {"o": o, "lse": lse}
