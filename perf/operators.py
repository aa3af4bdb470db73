"""The serving operators' cases: what each stands for, its inputs, its plain form and its value in 64 bits.

Four operators, used together by a decoder that serves many requests from one paged
key/value cache:

* prompt: causal attention of whole prompts, packed one after another, with grouped heads;
* paged:  new tokens (one or a chunk for each request) go into the pages of the cache and
          attend to everything cached for their request;
* select: one step of beam search: the best `beams` of beams x vocabulary candidates;
* reorder: the beams' cached states follow their parents.

Types: "f32" (inputs, cache and output in f32), "bf16" (all bf16), "mixed" (q, k and v in f32
as the int8 projections write them, cache and output in bf16).
"""
import itertools
import math
import random

import torch

own = False

F32, BF16 = torch.float32, torch.bfloat16
DEV = "cuda"


# ---- the cases ----------------------------------------------------------------------------------


def _text(v):
    return ",".join(str(int(x)) for x in v)


def _ints(s):
    return [int(x) for x in s.split(",")]


def _spread(n, lo, hi, seed):
    """n lengths between lo and hi, spread over their logarithm, both ends among them."""
    r = random.Random(seed)
    v = [int(math.exp(r.uniform(math.log(lo), math.log(hi)))) for _ in range(n)]
    v[0], v[n // 2] = lo, hi
    return v


def listed():
    return [
        # a few short requests reach a GPT-2 small server together: latency
        {"name": "prompt_short", "op": "prompt", "type": "mixed", "heads": 12, "kv_heads": 12, "dim": 64,
         "lens": "7,33,1,19"},
        # a batch of prompts of a GPT-2 XL in fp32 mode, up to its 1024 positions
        {"name": "prompt_xl_f32", "op": "prompt", "type": "f32", "heads": 25, "kv_heads": 25, "dim": 64,
         "lens": "1024,700,333,1019"},
        # one long prompt, heads in groups of four
        {"name": "prompt_long", "op": "prompt", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "lens": "8192"},
        # one user of a GPT-2 small in fp32 mode, one token at a time: latency
        {"name": "decode_one", "op": "paged", "type": "f32", "heads": 12, "kv_heads": 12, "dim": 64,
         "page": 16, "new": "1", "lens": "301"},
        # sixteen users of a GPT-2 small whose cache is held in bf16
        {"name": "decode_batch", "op": "paged", "type": "mixed", "heads": 12, "kv_heads": 12, "dim": 64,
         "page": 32, "new": _text([1] * 16), "lens": _text(_spread(16, 20, 1024, 1))},
        # a full server: 64 requests of very different lengths, grouped heads, one token each
        {"name": "decode_full", "op": "paged", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "new": _text([1] * 64), "lens": _text(_spread(64, 100, 8192, 2))},
        # prompts taken in chunks beside requests that decode and one that waits
        {"name": "chunk_mixed_batch", "op": "paged", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "new": "512,1,130,0,257,64", "lens": "4608,8000,130,77,1025,8192"},
        # follow-up turns of a GPT-2 XL in fp32 mode
        {"name": "chunk_xl_f32", "op": "paged", "type": "f32", "heads": 25, "kv_heads": 25, "dim": 64,
         "page": 16, "new": "64,17,128,1", "lens": "1000,17,512,801"},
        # four beams of one request over GPT-2's vocabulary
        {"name": "select_one", "op": "select", "requests": 1, "beams": 4, "vocab": 50257},
        # a full server of beam searches
        {"name": "select_full", "op": "select", "requests": 64, "beams": 8, "vocab": 50257},
        # the step's cache moves for one request of a GPT-2 small in fp32 mode
        {"name": "reorder_one", "op": "reorder", "type": "f32", "layers": 12, "kv_heads": 12, "dim": 64,
         "page": 16, "beams": 4, "prompt": "25", "lens": "58"},
        # and for sixteen requests of eight beams with a bf16 cache
        {"name": "reorder_full", "op": "reorder", "type": "bf16", "layers": 12, "kv_heads": 12, "dim": 64,
         "page": 64, "beams": 8, "prompt": _text(_spread(16, 5, 900, 3)),
         "lens": _text([p + n for p, n in zip(_spread(16, 5, 900, 3), _spread(16, 1, 100, 4))])},
    ]


_HEADS = [(12, 12, 64), (25, 25, 64), (32, 8, 128), (16, 2, 128), (6, 2, 80), (8, 1, 64), (20, 4, 96), (4, 4, 32),
          (16, 16, 128)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "paged", "paged", "paged", "select", "reorder"])
    heads, kv_heads, dim = rng.choice(_HEADS)
    kind = rng.choice(["f32", "bf16", "mixed"])
    page = rng.choice([16, 32, 64, 128])
    if op == "prompt":
        n = _log(rng, 1, 12)
        # every request costs up to top^2: together no more than the longest listed prompt
        top = int(8192 * math.sqrt(32 * 128 / (max(heads, 32) * 128 * n)))
        if kind == "f32":
            top = min(top, 2048)
        lens = [_log(rng, 1, top) for _ in range(n)]
        return {"op": op, "type": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "lens": _text(lens)}
    if op == "paged":
        chunk = rng.random() < 0.5
        n = _log(rng, 1, 12 if chunk else 64)
        top = int(min(8192, 64 * 2048 * 8 * 128 / (n * kv_heads * dim * (2 if kind == "f32" else 1))))
        lens = [_log(rng, 1, top) for _ in range(n)]
        new = [rng.choice([0, 1, _log(rng, 1, 512), _log(rng, 1, 512)]) if chunk else 1 for _ in range(n)]
        new = [min(a, b) for a, b in zip(new, lens)]
        if sum(new) == 0:
            new[0] = 1
        return {"op": op, "type": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
                "new": _text(new), "lens": _text(lens)}
    if op == "select":
        beams = rng.randint(1, 16)
        vocab = rng.choice([50257, _log(rng, 40, 64000)])
        n = _log(rng, 1, max(1, 64 * 8 * 50257 // (beams * vocab)) if beams * vocab * 64 > 64 * 8 * 50257 else 64)
        return {"op": op, "requests": n, "beams": beams, "vocab": vocab}
    beams = rng.randint(1, 12)
    n = _log(rng, 1, 16)
    prompt = [_log(rng, 1, 900) for _ in range(n)]
    lens = [p + rng.randint(1, 100) for p in prompt]
    size = 4 if kind == "f32" else 2
    token = 4 * kv_heads * dim * size  # one token of one layer, read and written
    layers = max(1, min(48, 250_000_000 // (token * beams * sum(m % page for m in lens) + 1)))
    layers = _log(rng, 1, layers)
    return {"op": op, "type": "f32" if kind == "f32" else "bf16", "layers": layers, "kv_heads": kv_heads, "dim": dim,
            "page": page, "beams": beams, "prompt": _text(prompt), "lens": _text(lens)}


def work(case):
    op = case["op"]
    if op == "select":
        rows = case["requests"] * case["beams"]
        return {"bytes": rows * (4 * case["vocab"] + 4 + 1 + 4 + 4 + 4 + 1), "flops": 4 * rows * case["vocab"]}
    size = 4 if case["type"] == "f32" else 2
    lens = _ints(case["lens"])
    if op == "reorder":
        # a beam that keeps its state costs nothing; one in four or so does: all of them are counted
        token = 2 * case["layers"] * case["kv_heads"] * case["dim"] * size
        moved = sum(case["beams"] * (n % case["page"]) for n in lens)
        pages = sum(case["beams"] * -(-n // case["page"]) for n in lens)
        return {"bytes": 2 * moved * token + 8 * pages, "flops": 0}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    x = 2 if case["type"] == "bf16" else 4
    new = _ints(case["new"]) if op == "paged" else lens
    rows = sum(new)
    pairs = sum(m * n - m * (m - 1) // 2 for m, n in zip(new, lens))
    moved = rows * (heads * dim * (x + size) + 2 * kv_heads * dim * x)
    if op == "paged":
        moved += 2 * kv_heads * dim * size * (sum(n for m, n in zip(new, lens) if m) + rows)
        moved += sum(4 * -(-n // case["page"]) for n in lens)
    return {"bytes": moved, "flops": 4 * heads * dim * pairs}


# ---- inputs -------------------------------------------------------------------------------------


def _types(kind):
    return (BF16 if kind == "bf16" else F32), (F32 if kind == "f32" else BF16)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cu(lens):
    return _i32([0, *itertools.accumulate(lens)])


def _projected(case, rows, gen):
    """q, k and v as views of one projection's rows (q | k | v), as the decoder has them."""
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    x = torch.randn((rows, (heads + 2 * kv_heads) * dim), generator=gen, device=DEV)
    x[:, : heads * dim] *= 1.5  # attention that prefers some keys
    x = x.to(_types(case["type"])[0])
    q, k, v = x.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1)
    return q.view(rows, heads, dim), k.view(rows, kv_heads, dim), v.view(rows, kv_heads, dim)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    rng = random.Random(int(seed))
    op = case["op"]
    s = {"op": op}
    if op == "select":
        n, w, vocab = case["requests"], case["beams"], case["vocab"]
        logits = torch.randn((n * w, vocab), generator=gen, device=DEV)
        logits = logits * 2.0 + 4.0 * torch.rand((n * w, vocab), generator=gen, device=DEV).pow(6)
        scores = -12.0 * torch.rand((n, w), generator=gen, device=DEV)
        scores[:, 1:][torch.rand((n, w - 1), generator=gen, device=DEV) < 0.04] = -math.inf  # beams not begun
        done = (torch.rand((n, w), generator=gen, device=DEV) < 0.1).to(torch.uint8)
        s.update(logits=logits, scores=scores, done=done, eos=vocab - 1)
        return s
    lens = _ints(case["lens"])
    if op == "prompt":
        s["q"], s["k"], s["v"] = _projected(case, sum(lens), gen)
        s.update(cu=_cu(lens), top=max(lens))
        s["out_type"] = _types(case["type"])[1]
        return s
    page, kv_heads, dim = case["page"], case["kv_heads"], case["dim"]
    cache = _types(case["type"])[1]
    if op == "paged":
        new = _ints(case["new"])
        s["q"], s["k"], s["v"] = _projected(case, sum(new), gen)
        width = -(-max(lens) // page)
        used = [-(-n // page) for n in lens]
        order = list(range(sum(used) + 3))
        rng.shuffle(order)
        table = [[order.pop() for _ in range(u)] + [0] * (width - u) for u in used]
        shape = (sum(used) + 3, kv_heads, page, dim)
        s["k_pages"] = torch.randn(shape, generator=gen, device=DEV, dtype=cache)
        s["v_pages"] = torch.randn(shape, generator=gen, device=DEV, dtype=cache)
        s.update(table=_i32(table), lens=_i32(lens), cu=_cu(new), top=max(new))
        return s
    # reorder: the beams of a request share its prompt's full pages and own the later ones
    w, prompt = case["beams"], _ints(case["prompt"])
    width = max(-(-(n + page) // page) for n in lens)
    rows, count = [], 0
    for p in prompt:
        shared = list(range(count, count + p // page))
        count += len(shared)
        for _ in range(w):
            rows.append(shared + list(range(count, count + width - len(shared))))
            count += width - len(shared)
    owned = _i32(rows)
    shape = (case["layers"], count, kv_heads, page, dim)
    s["k_pages"] = torch.randn(shape, generator=gen, device=DEV, dtype=cache)
    s["v_pages"] = torch.randn(shape, generator=gen, device=DEV, dtype=cache)
    # what earlier steps left in the tables: full pages of any beam of the request
    table = [list(r) for r in rows]
    for b, n in enumerate(lens):
        for i in range(w):
            for p in range(n // page):
                table[b * w + i][p] = rows[b * w + rng.randrange(w)][p]
    parent = [[min(int(rng.random() ** 2 * w), w - 1) if rng.random() < 0.75 else i for i in range(w)] for _ in lens]
    s.update(parent=_i32(parent), table=_i32(table), owned=owned, lens=_i32(lens))
    return s


# ---- the plain forms ----------------------------------------------------------------------------


def _softmax_product(scores, seen, v):
    """softmax over the keys that are seen, times v; a row that sees none gives zeros."""
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    weight = scores.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    return (weight @ v) / torch.where(total == 0, torch.ones_like(total), total)


def _attend(q, k, v, cu, top, lens, out_type):
    """q [T, H, D] packed rows; k and v [B, KV, N, D] each request's keys, lens [B] of them its own."""
    heads, dim = q.shape[1:]
    n, kv_heads, keys = k.shape[:3]
    at = torch.arange(top, device=DEV)
    new = (cu[1:] - cu[:-1]).long()
    row = cu[:-1, None].long() + at
    live = at < new[:, None]
    x = q[torch.where(live, row, torch.zeros_like(row))].float()  # [B, top, H, D]
    x = x.view(n, top, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4).reshape(n, kv_heads, -1, dim)
    j = torch.arange(keys, device=DEV)
    held = j < lens[:, None]
    k = torch.where(held[:, None, :, None], k.float(), torch.zeros((), device=DEV))
    v = torch.where(held[:, None, :, None], v.float(), torch.zeros((), device=DEV))
    scores = (x @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(dim))
    seen = j <= (lens[:, None].long() - new[:, None] + at)[:, :, None]
    seen = (seen & held[:, None, :])[:, None, None]
    y = _softmax_product(scores.view(n, kv_heads, -1, top, keys), seen, v[:, :, None])
    y = y.permute(0, 3, 1, 2, 4).reshape(n, top, heads, dim)
    out = torch.zeros(q.shape, dtype=out_type, device=DEV)
    out[row[live]] = y[live].to(out_type)
    return out


def _plain_prompt(s):
    lens = s["cu"][1:] - s["cu"][:-1]
    at = torch.arange(s["top"], device=DEV)
    row = s["cu"][:-1, None].long() + at
    row = torch.where(at < lens[:, None], row, torch.zeros_like(row))
    k, v = s["k"][row].transpose(1, 2), s["v"][row].transpose(1, 2)
    # what the cache type holds of k and v
    k, v = k.to(s["out_type"]), v.to(s["out_type"])
    return {"out": _attend(s["q"], k, v, s["cu"], s["top"], lens, s["out_type"])}


def _plain_paged(s):
    kp, vp = s["k_pages"], s["v_pages"]
    page = kp.shape[2]
    n = s["lens"].numel()
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    rows = torch.arange(s["q"].shape[0], device=DEV)
    b = torch.searchsorted(s["cu"][1:].long(), rows, right=True)
    place = s["lens"].long()[b] - new[b] + rows - s["cu"].long()[b]
    where = s["table"].long()[b, place // page]
    kp[where, :, place % page] = s["k"].to(kp.dtype)
    vp[where, :, place % page] = s["v"].to(vp.dtype)
    table = s["table"].long()
    k = kp[table].transpose(1, 2).reshape(n, kp.shape[1], -1, kp.shape[3])
    v = vp[table].transpose(1, 2).reshape(n, kp.shape[1], -1, kp.shape[3])
    return {"out": _attend(s["q"], k, v, s["cu"], s["top"], s["lens"], kp.dtype), "k": kp, "v": vp}


def _plain_select(s):
    n, w = s["scores"].shape
    x = s["logits"].view(n, w, -1)
    vocab = x.shape[2]
    x = torch.where(x.isnan(), torch.full((), -math.inf, device=DEV), x)
    top = x.amax(-1, keepdim=True)
    lse = top + (x - top).exp().sum(-1, keepdim=True).log()
    total = s["scores"][:, :, None] + (x - lse)
    total = torch.where(total.isnan(), torch.full((), -math.inf, device=DEV), total)
    ends = torch.arange(vocab, device=DEV) == s["eos"]
    kept = torch.where(ends, s["scores"][:, :, None], torch.full((), -math.inf, device=DEV))
    total = torch.where(s["done"][:, :, None] != 0, kept, total).view(n, -1)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :w], at[:, :w]
    parent, token = at // vocab, at % vocab
    done = (torch.gather(s["done"], 1, parent) != 0) | (token == s["eos"])
    return {"scores": best, "parent": parent.int(), "token": token.int(), "done": done.to(torch.uint8)}


def _plain_reorder(s):
    n, w = s["parent"].shape
    kp, vp, table, owned = s["k_pages"], s["v_pages"], s["table"], s["owned"].long()
    page = kp.shape[3]
    full, rest = (s["lens"].long() // page).repeat_interleave(w), (s["lens"].long() % page).repeat_interleave(w)
    source = (torch.arange(n, device=DEV)[:, None] * w + s["parent"].long()).view(-1)
    into = owned.gather(1, full[:, None])[:, 0]
    moved = (torch.arange(page, device=DEV) < rest[:, None])[None, :, None, :, None]
    kp[:, into] = torch.where(moved, kp[:, into[source]], kp[:, into])
    vp[:, into] = torch.where(moved, vp[:, into[source]], vp[:, into])
    column = torch.arange(table.shape[1], device=DEV)
    table.copy_(torch.where(column < full[:, None], table[source], owned.int()))
    return {"table": table, "k": kp, "v": vp}


def run(s):
    op = s["op"]
    if not own:
        return {"prompt": _plain_prompt, "paged": _plain_paged, "select": _plain_select, "reorder": _plain_reorder}[op](s)
    from mini_tensorrt_b200 import serving
    if op == "prompt":
        return {"out": serving.prompt_attention(s["q"], s["k"], s["v"], s["cu"], out_dtype=s["out_type"])}
    if op == "paged":
        out = serving.paged_attention(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cu"])
        return {"out": out, "k": s["k_pages"], "v": s["v_pages"]}
    if op == "select":
        scores, parent, token, done = serving.beam_select(s["logits"], s["scores"], s["done"], s["eos"])
        return {"scores": scores, "parent": parent, "token": token, "done": done}
    serving.beam_reorder(s["parent"], s["table"], s["owned"], s["lens"], s["k_pages"], s["v_pages"])
    return {"table": s["table"], "k": s["k_pages"], "v": s["v_pages"]}


# ---- in 64 bits ---------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "select":
        n, w, vocab = case["requests"], case["beams"], case["vocab"]
        total = s["scores"].double()[:, :, None] + torch.log_softmax(s["logits"].double().view(n, w, vocab), dim=2)
        for b, i in s["done"].nonzero().tolist():
            total[b, i] = -math.inf
            total[b, i, s["eos"]] = s["scores"][b, i].double()
        best = total.view(n, -1).topk(w, dim=1).values
        return {"scores": best, "parent": None, "token": None, "done": None}
    if op == "reorder":
        w, page = case["beams"], case["page"]
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        for b, n in enumerate(_ints(case["lens"])):
            mine = s["owned"][b * w:(b + 1) * w, n // page].tolist()
            for i, j in enumerate(s["parent"][b].tolist()):
                for to, come in ((kp, s["k_pages"]), (vp, s["v_pages"])):
                    to[:, mine[i], :, : n % page] = come[:, mine[j], :, : n % page].double()
        return {"table": None, "k": kp, "v": vp}

    def last_rows(q, k, v):
        """The last rows of a request: q [m, H, D] against k and v [n, KV, D], row i seeing n - m + i + 1 keys."""
        m, heads, dim = q.shape
        n, kv_heads, _ = k.shape
        out = torch.empty((m, heads, dim), dtype=torch.float64, device=DEV)
        limit = torch.arange(n - m, n, device=DEV)[:, None]
        hidden = torch.arange(n, device=DEV)[None, :] > limit
        for h in range(heads):
            g = h // (heads // kv_heads)
            p = torch.einsum("md,nd->mn", q[:, h].double(), k[:, g].double()) / math.sqrt(dim)
            p[hidden] = -math.inf
            p = torch.softmax(p, dim=1)
            out[:, h] = p @ v[:, g].double()
        return out

    lens = _ints(case["lens"])
    held = _types(case["type"])[1]
    out, at = [], 0
    if op == "prompt":
        for n in lens:
            r = slice(at, at + n)
            out.append(last_rows(s["q"][r], s["k"][r].to(held), s["v"][r].to(held)))
            at += n
        return {"out": torch.cat(out)}
    page = case["page"]
    kp, vp = s["k_pages"], s["v_pages"]
    for b, (m, n) in enumerate(zip(_ints(case["new"]), lens)):
        for i in range(m):
            place = n - m + i
            where = int(s["table"][b, place // page])
            kp[where, :, place % page] = s["k"][at + i].to(held)
            vp[where, :, place % page] = s["v"][at + i].to(held)
        pages = s["table"][b, : -(-n // page)].long()
        k = kp[pages].permute(0, 2, 1, 3).flatten(0, 1)[:n]
        v = vp[pages].permute(0, 2, 1, 3).flatten(0, 1)[:n]
        if m:
            out.append(last_rows(s["q"][at:at + m], k, v))
        at += m
    return {"out": torch.cat(out), "k": kp.double(), "v": vp.double()}
