"""Cases for the paged KV-cache operators and the logits operator: inputs, plain forms, work and 64-bit answers.

Four operators of one serving step: append (rotary positions, K and V written to pages), attend (one new token per
sequence over its pages, optionally adding each position's attention weight to its mass), evict (the heaviest
positions copied to fresh pages) and logits (penalties, biases, grammar mask, greedy token)."""
import math
import os
import random
import sys

import numpy
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
KV_TYPES = {"f32": 0, "f16": 1, "bf16": 2}
ROPE_BASE = 5000000.0


def listed():
    model = {"heads": 16, "kv_heads": 2, "dim": 128}
    return [
        # the smallest call: one conversation that has just begun, fp32 cache as the engine's default
        dict(model, name="attend one short", op="attend", kv="f32", page=16, seqs=1, len_min=137, len_max=137, mass=False, holes=False, split=False),
        # one conversation after an 8192-position prefill
        dict(model, name="attend one 8k", op="attend", kv="f32", page=64, seqs=1, len_min=8193, len_max=8193, mass=False, holes=False, split=False),
        # a full batch of 64 conversations of unlike lengths that will be evicted from: weights are accumulated
        dict(model, name="attend 64 ragged mass", op="attend", kv="f16", page=16, seqs=64, len_min=300, len_max=4096, mass=True, holes=False, split=False),
        # a few very long documents
        dict(model, name="attend 4 of 128k", op="attend", kv="f16", page=64, seqs=4, len_min=131072, len_max=131072, mass=False, holes=False, split=False),
        # groups of three heads, pages that end inside a tile, absent pages, empty rows, head-major pool
        dict(name="attend odd bf16", op="attend", heads=12, kv_heads=4, dim=64, kv="bf16", page=24, seqs=48, len_min=1, len_max=3001, mass=True, holes=True, split=True),
        # one decode step of 64 conversations
        dict(model, name="append 64 tokens", op="append", kv="f16", page=16, seqs=64, tokens=64, split=False),
        # a prompt of 8192 positions
        dict(model, name="append prompt 8k", op="append", kv="f32", page=64, seqs=1, tokens=8192, split=False),
        # one conversation that went a page over its budget
        dict(model, name="evict one page", op="evict", kv="f32", page=64, seqs=1, len=2112, keep=2048, sink=4, recent=256, split=False),
        # a batch cut to half
        dict(model, name="evict 64 to half", op="evict", kv="f16", page=16, seqs=64, len=4096, keep=2048, sink=4, recent=512, split=False),
        # one long document compressed to a quarter, an odd length and an odd page
        dict(model, name="evict long to quarter", op="evict", kv="bf16", page=24, seqs=1, len=65537, keep=16384, sink=16, recent=2048, split=True),
        # one conversation's logits
        dict(name="logits one", op="logits", vocab=130560, seqs=1, hist=300, bias=0, mask=False),
        # a batch with long histories, user biases and grammars
        dict(name="logits 64", op="logits", vocab=130560, seqs=64, hist=4096, bias=64, mask=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "evict", "logits"])
    if op == "logits":
        return {"op": op, "vocab": _log(rng, 8000, 260000), "seqs": _log(rng, 1, 64), "hist": _log(rng, 1, 8192),
                "bias": rng.choice([0, 1, 17, 300]), "mask": rng.random() < 0.5}
    heads, kv_heads, dim = rng.choice([(16, 2, 128), (16, 2, 128), (12, 4, 64), (8, 8, 64), (16, 1, 128), (20, 4, 128), (32, 4, 64)])
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "kv": rng.choice(["f32", "f16", "bf16"]),
         "page": rng.choice([16, 16, 64, 128, 24, 7, 1]), "split": rng.random() < 0.3}
    row = kv_heads * dim * SIZES[c["kv"]]   # bytes of K of one position
    if op == "append":
        return {**c, "seqs": _log(rng, 1, 32), "tokens": min(_log(rng, 1, 16384), (8192 * 1024) // row)}
    most = (131072 * 4 * 512) // row // (4 if op == "evict" else 2)   # positions in all
    n = _log(rng, 1, 64)
    top = max(2, min(131072 if op == "attend" else 65537, most // n))
    if op == "evict":
        length = max(33, min(top, _log(rng, 65, 65537)))
        keep = max(8, int(length * rng.uniform(0.2, 0.97)))
        return {**c, "seqs": n, "len": length, "keep": keep, "sink": min(4, keep // 2), "recent": keep // rng.choice([3, 8, 50])}
    hi = min(top, _log(rng, 1, 131072))
    return {**c, "seqs": n, "len_min": max(1, hi // rng.choice([1, 4, 20])), "len_max": hi, "mass": rng.random() < 0.5, "holes": rng.random() < 0.3}


def _lengths(case):
    """Lengths of the sequences: a property of the case, not of its seed."""
    r = random.Random(case["seqs"] * 1000003 + case["len_max"])
    got = [case["len_max"]] + [r.randint(case["len_min"], case["len_max"]) for _ in range(case["seqs"] - 1)]
    if case["holes"]:
        got = [0 if i % 7 == 3 else n for i, n in enumerate(got)]
    return got


def _absent(case, seq, page):
    """Pages that a sequence has given back; its row 5 has none left."""
    return case["holes"] and (seq == 5 or (seq * 31 + page * 17) % 11 == 4)


def _positions(case):
    """Positions that each sequence still has."""
    got = []
    for s, n in enumerate(_lengths(case)):
        pages = -(-n // case["page"])
        got.append(n if not case["holes"] else sum(min(case["page"], n - p * case["page"]) for p in range(pages) if not _absent(case, s, p)))
    return got


def work(case):
    if case["op"] == "logits":
        n, v = case["seqs"], case["vocab"]
        return {"bytes": n * (8 * v + 4 * case["hist"] + 8 * case["bias"] + (v // 8 if case["mask"] else 0) + 4), "flops": 4 * n * v}
    d, hq, hk, e = case["dim"], case["heads"], case["kv_heads"], SIZES[case["kv"]]
    if case["op"] == "append":
        t = case["tokens"]
        return {"bytes": t * (2 * hq * d * 4 + 2 * hk * d * (4 + e) + d * 4 + hk * 4), "flops": 3 * t * (hq + hk) * d}
    if case["op"] == "evict":
        n, keep = case["seqs"], min(case["keep"], case["len"])
        return {"bytes": n * hk * (4 * case["len"] + keep * (4 * d * e + 12)), "flops": n * hk * case["len"]}
    t = sum(_positions(case))
    return {"bytes": t * hk * (2 * d * e + (8 if case["mass"] else 0)) + case["seqs"] * hq * d * 8, "flops": 4 * t * hq * d}


# ---------------------------------------------------------------- inputs
def _engine():
    """The framework's Python binding, whose folder is not a package name."""
    at = os.path.join(os.getcwd(), "minicpm5.cpp_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from mcpm import engine
    return engine


def _pool(case, pages, g):
    """Pool of K or V, indexed [page][slot][KV head][dim]; split: the heads of a page lie apart in memory."""
    n, h, d = case["page"], case["kv_heads"], case["dim"]
    x = torch.randn((pages, h, n, d) if case["split"] else (pages, n, h, d), device="cuda", generator=g).to(TYPES[case["kv"]])
    return x.transpose(1, 2) if case["split"] else x


def _geometry(s, case, pages, cols):
    """The descriptors that a program keeps beside its pools."""
    E = _engine()
    k = s["k"]
    s["E"] = E
    s["cfg"] = E.paged_config(KV_TYPES[case["kv"]], case["heads"], case["kv_heads"], case["dim"], case["page"], pages, case["seqs"], cols,
                              k.stride(0), k.stride(1), k.stride(2))
    s["pool"] = E.paged_pool(k.data_ptr(), s["v"].data_ptr(), s["mass"].data_ptr() if s["mass"] is not None else 0)
    s["workspace"] = torch.zeros(E.paged_workspace_bytes(s["cfg"]), dtype=torch.uint8, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "logits":
        n, v = case["seqs"], case["vocab"]
        s["logits"] = 3.0 * torch.randn((n, v), device="cuda", generator=g)
        # tokens repeat: low ids are frequent
        s["hist"] = (v * torch.rand((n, case["hist"]), device="cuda", generator=g) ** 3).to(torch.int32).clamp_(0, v - 1)
        s["hist_len"] = torch.tensor([case["hist"] - (i * case["hist"]) // (2 * n) for i in range(n)], dtype=torch.int32, device="cuda")
        s["penalties"] = torch.rand((n, 3), device="cuda", generator=g) * torch.tensor([0.5, 0.3, 0.6], device="cuda") + torch.tensor([1.0, 0.0, 0.0], device="cuda")
        s["bias_token"] = torch.randint(0, v, (n, max(1, case["bias"])), device="cuda", generator=g, dtype=torch.int32)
        s["bias"] = 4.0 * torch.randn((n, max(1, case["bias"])), device="cuda", generator=g)
        s["bias_len"] = torch.full((n,), case["bias"], dtype=torch.int32, device="cuda")
        # a grammar allows a part of the vocabulary
        s["allow"] = torch.randint(-2 ** 31, 2 ** 31, (n, (v + 31) // 32), device="cuda", generator=g, dtype=torch.int32) if case["mask"] else None
        s["out"], s["token"] = torch.empty_like(s["logits"]), torch.empty(n, dtype=torch.int32, device="cuda")
        if own:
            E = _engine()
            s["E"] = E
        return s
    page, n = case["page"], case["seqs"]
    if case["op"] == "append":
        per = -(-case["tokens"] // n)
        lens = [min(per, max(0, case["tokens"] - i * per)) for i in range(n)]
    else:
        lens = _lengths(case) if case["op"] == "attend" else [case["len"]] * n
    want = [-(-x // page) for x in lens]
    keep = -(-case["keep"] // page) if case["op"] == "evict" else 0
    cols, pages = max(1, max(want)), sum(want) + n * keep + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).cpu()
    table, at = torch.full((n, cols), -1, dtype=torch.int32), 0
    for i, w in enumerate(want):
        table[i, :w] = order[at:at + w]
        at += w
    if case["op"] == "attend" and case["holes"]:
        for i, w in enumerate(want):
            for p in range(w):
                if _absent(case, i, p):
                    table[i, p] = -1
    s["table"], s["k"], s["v"] = table.cuda(), _pool(case, pages, g), _pool(case, pages, g)
    s["len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["mass"] = None
    if case["op"] != "attend" or case["mass"]:
        # accumulated weights are small with a heavy tail
        s["mass"] = torch.rand((pages, case["kv_heads"], page), device="cuda", generator=g) ** 6 * 5.0
    if case["op"] == "evict":
        dst = torch.full((n, cols), -1, dtype=torch.int32)
        for i in range(n):
            dst[i, :keep] = order[at:at + keep]
            at += keep
        s["dst"] = dst.cuda()
        s["new_len"] = torch.empty(n, dtype=torch.int32, device="cuda")
        s["kept"] = torch.empty((n, case["kv_heads"], case["keep"]), dtype=torch.int32, device="cuda")
    elif case["op"] == "attend":
        s["q"] = 1.5 * torch.randn((n, case["heads"] * case["dim"]), device="cuda", generator=g)
        s["out"] = torch.empty_like(s["q"])
    else:
        t, d = case["tokens"], case["dim"]
        s["qkv"] = torch.randn((t, (case["heads"] + 2 * case["kv_heads"]) * d), device="cuda", generator=g)   # one projection's output
        s["q_out"] = torch.empty((t, case["heads"] * d), device="cuda")
        slot = torch.cat([torch.arange(x, dtype=torch.int32) for x in lens])
        s["tok_slot"], s["tok_seq"] = slot.cuda(), torch.cat([torch.full((x,), i, dtype=torch.int32) for i, x in enumerate(lens)]).cuda()
        s["tok_pos"] = s["tok_slot"] + 5   # a cache that was evicted from: positions run ahead of slots
        angle = torch.arange(max(lens) + 6, dtype=torch.float64)[:, None] * ROPE_BASE ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).float().cuda()
    if own:
        _geometry(s, case, pages, cols)
    return s


# ---------------------------------------------------------------- plain forms
def _slots(s, table, cols):
    """(pages, slots, visible) of positions 0 .. cols - 1 of every sequence."""
    page, pages = s["case"]["page"], s["k"].shape[0]
    j = torch.arange(cols, device="cuda")
    p = table[:, (j // page).clamp(max=table.shape[1] - 1)].long()
    seen = (p >= 0) & (p < pages)
    return p.clamp(0, pages - 1), (j % page).expand_as(p), seen


def _plain_attend(s):
    c = s["case"]
    n, h, d = c["seqs"], c["kv_heads"], c["dim"]
    cols = min(s["table"].shape[1] * c["page"], c["len_max"])
    page, slot, seen = _slots(s, s["table"], cols)
    seen = seen & (torch.arange(cols, device="cuda")[None] < s["len"][:, None])
    q = s["q"].view(n, h, -1, d)
    k = s["k"][page, slot].float()                                       # [seqs, positions, KV heads, dim]
    score = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))   # [seqs, KV heads, group, positions]
    del k
    score = score.masked_fill(~seen[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = (score - torch.where(top == -math.inf, 0.0, top)).exp()
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    v = s["v"][page, slot].float().masked_fill(~seen[:, :, None, None], 0.0)
    out = torch.matmul(p, v.permute(0, 2, 1, 3)).reshape(n, -1)
    if s["mass"] is None:
        return {"out": out}
    row, col = seen.nonzero(as_tuple=True)
    at, to = page[row, col], slot[row, col]
    s["mass"][at, :, to] += p.sum(2)[row, :, col]
    return {"out": out, "mass": s["mass"]}


def _plain_append(s):
    c = s["case"]
    t, d, hq, hk = c["tokens"], c["dim"], c["heads"], c["kv_heads"]
    q, k, v = s["qkv"].view(t, -1, d).split([hq, hk, hk], 1)
    cos, sin = s["rope"][s["tok_pos"].long()].unbind(-1)

    def turn(x):
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([cos[:, None] * a - sin[:, None] * b, sin[:, None] * a + cos[:, None] * b], -1).flatten(-2)

    slot = s["tok_slot"].long()
    page = s["table"][s["tok_seq"].long(), slot // c["page"]].long()
    s["k"][page, slot % c["page"]] = turn(k).to(s["k"].dtype)
    s["v"][page, slot % c["page"]] = v.to(s["v"].dtype)
    s["mass"][page, :, slot % c["page"]] = 0.0
    return {"q": turn(q).reshape(t, -1), "k": s["k"], "v": s["v"], "mass": s["mass"]}


def _plain_evict(s):
    c = s["case"]
    n, h, length, keep = c["seqs"], c["kv_heads"], c["len"], min(c["keep"], c["len"])
    page, slot, _ = _slots(s, s["table"], length)
    mass = s["mass"][page, :, slot].transpose(1, 2)                      # [seqs, KV heads, positions]
    j = torch.arange(length, device="cuda")
    held = (j < c["sink"]) | (j >= length - c["recent"])
    order = mass.masked_fill(held, math.inf).sort(dim=-1, descending=True, stable=True).indices
    kept = order[..., :keep].sort(-1).values                             # [seqs, KV heads, keep]
    to, place, _ = _slots(s, s["dst"], keep)
    row, head = torch.arange(n, device="cuda")[:, None, None], torch.arange(h, device="cuda")[None, :, None]
    a, b, x, y = page[row, kept], slot[row, kept], to[:, None], place[:, None]
    s["k"][x, y, head] = s["k"][a, b, head]
    s["v"][x, y, head] = s["v"][a, b, head]
    s["mass"][x, head, y] = s["mass"][a, head, b]
    new_len = torch.full((n,), keep, dtype=torch.int32, device="cuda")
    return {"k": s["k"], "v": s["v"], "mass": s["mass"], "kept": kept.to(torch.int32), "new_len": new_len}


def _plain_logits(s):
    c = s["case"]
    n, v = c["seqs"], c["vocab"]
    x = s["logits"]
    real = torch.arange(c["hist"], device="cuda")[None] < s["hist_len"][:, None]
    count = torch.zeros((n, v), device="cuda").scatter_add_(1, s["hist"].long(), real.float())
    rep, freq, pres = (p[:, None] for p in s["penalties"].unbind(1))
    x = torch.where(count > 0, torch.where(x > 0, x / rep, x * rep) - (freq * count + pres), x)
    if c["bias"]:
        # a token that is listed twice takes its last entry
        at = torch.full((n, v), -1, dtype=torch.int64, device="cuda")
        at.scatter_reduce_(1, s["bias_token"].long(), torch.arange(c["bias"], device="cuda").expand(n, -1), "amax")
        x = torch.where(at >= 0, x + s["bias"].gather(1, at.clamp(min=0)), x)
    if c["mask"]:
        t = torch.arange(v, device="cuda")
        x = x.masked_fill(((s["allow"][:, t // 32] >> (t % 32)) & 1) == 0, -math.inf)
    top = x.amax(1, keepdim=True)
    token = torch.where(x == top, torch.arange(v, device="cuda"), v).amin(1)
    return {"logits": x, "token": torch.where(top[:, 0] == -math.inf, -1, token).to(torch.int32)}


# ---------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if not own:
        return {"attend": _plain_attend, "append": _plain_append, "evict": _plain_evict, "logits": _plain_logits}[op](s)
    E, c = s["E"], s["case"]
    if op == "logits":
        n, v = c["seqs"], c["vocab"]
        more = {"allow": s["allow"].data_ptr(), "allow_stride": s["allow"].stride(0)} if c["mask"] else {}
        if c["bias"]:
            more.update(bias_token=s["bias_token"].data_ptr(), bias=s["bias"].data_ptr(), bias_stride=s["bias"].stride(0), bias_len=s["bias_len"].data_ptr())
        E.logits_process(s["logits"].data_ptr(), s["out"].data_ptr(), n, v, hist=s["hist"].data_ptr(), hist_stride=s["hist"].stride(0),
                         hist_len=s["hist_len"].data_ptr(), penalties=s["penalties"].data_ptr(), argmax=s["token"].data_ptr(), **more)
        return {"logits": s["out"], "token": s["token"]}
    if op == "attend":
        E.paged_attention(s["cfg"], s["pool"], s["table"].data_ptr(), s["len"].data_ptr(), c["seqs"], s["q"].data_ptr(), s["out"].data_ptr(),
                          s["workspace"].data_ptr(), s["workspace"].numel())
        return {"out": s["out"]} if s["mass"] is None else {"out": s["out"], "mass": s["mass"]}
    if op == "append":
        q, step = s["qkv"].data_ptr(), s["qkv"].stride(0)
        k = q + 4 * c["heads"] * c["dim"]
        E.paged_append(s["cfg"], s["pool"], s["table"].data_ptr(), c["tokens"], s["tok_slot"].data_ptr(), k, k + 4 * c["kv_heads"] * c["dim"],
                       tok_seq=s["tok_seq"].data_ptr(), tok_pos=s["tok_pos"].data_ptr(), q=q, q_out=s["q_out"].data_ptr(), q_stride=step, kv_stride=step,
                       rope=s["rope"].data_ptr(), rope_len=s["rope"].shape[0])
        return {"q": s["q_out"], "k": s["k"], "v": s["v"], "mass": s["mass"]}
    E.paged_evict(s["cfg"], s["pool"], s["table"].data_ptr(), s["len"].data_ptr(), s["dst"].data_ptr(), s["new_len"].data_ptr(), s["kept"].data_ptr(),
                  c["seqs"], c["keep"], c["sink"], c["recent"], s["workspace"].data_ptr(), s["workspace"].numel())
    return {"k": s["k"], "v": s["v"], "mass": s["mass"], "kept": s["kept"], "new_len": s["new_len"]}


# ---------------------------------------------------------------- 64-bit answers
def _rows(s, i, length, table=None):
    """(page, slot) of the present positions of sequence i, and those positions."""
    page = s["case"]["page"]
    ids = (s["table"] if table is None else table)[i].tolist()
    got = [(ids[j // page], j % page, j) for j in range(length) if ids[j // page] >= 0]
    return [torch.tensor(x, dtype=torch.int64, device="cuda") for x in zip(*got)] if got else None


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        rows = []
        for i in range(case["seqs"]):
            x = s["logits"][i].double()
            n = int(s["hist_len"][i])
            count = torch.bincount(s["hist"][i, :n].long(), minlength=case["vocab"]).double()
            rep, freq, pres = s["penalties"][i].double().tolist()
            hit = count > 0
            x[hit] = torch.where(x[hit] > 0, x[hit] / rep, x[hit] * rep) - freq * count[hit] - pres
            last = dict(zip(s["bias_token"][i, :case["bias"]].tolist(), s["bias"][i, :case["bias"]].double().tolist()))
            if last:
                x[torch.tensor(list(last), device="cuda")] += torch.tensor(list(last.values()), dtype=torch.float64, device="cuda")
            if case["mask"]:
                bits = (s["allow"][i].view(torch.uint8)[:, None] >> torch.arange(8, device="cuda", dtype=torch.uint8)) & 1   # little-endian words
                x[bits.reshape(-1)[:case["vocab"]] == 0] = -math.inf
            rows.append(x)
        return {"logits": torch.stack(rows), "token": None}
    n, h, d = case["seqs"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        x = s["qkv"].double().view(case["tokens"], -1, d)
        z = torch.view_as_complex(x.view(*x.shape[:2], d // 2, 2).contiguous())
        turned = torch.view_as_real(z * torch.view_as_complex(s["rope"].double())[s["tok_pos"].long()][:, None]).reshape(x.shape)
        k, v, mass = s["k"].double(), s["v"].double(), s["mass"].double()
        at = 0
        for i, length in enumerate(s["len"].tolist()):
            where = _rows(s, i, length)
            if where:
                k[where[0], where[1]] = turned[at:at + length, case["heads"]:case["heads"] + h]
                v[where[0], where[1]] = x[at:at + length, case["heads"] + h:]
                mass[where[0], :, where[1]] = 0.0
            at += length
        return {"q": turned[:, :case["heads"]].reshape(case["tokens"], -1), "k": k, "v": v, "mass": mass}
    if case["op"] == "evict":
        k, v, mass = s["k"].double(), s["v"].double(), s["mass"].double()
        for i in range(n):
            page, slot, j = _rows(s, i, case["len"])
            to = _rows(s, i, case["keep"], s["dst"])
            held = ((j < case["sink"]) | (j >= case["len"] - case["recent"])).cpu().numpy()
            for a in range(h):
                m = s["mass"][page, a, slot].cpu().numpy()
                free = (~held).nonzero()[0]
                room = min(case["keep"], case["len"]) - int(held.sum())
                # sorted by (-mass, position)
                best = free[(-m[free]).argsort(kind="stable")][:room]
                kept = torch.from_numpy(numpy.sort(numpy.concatenate([held.nonzero()[0], best]))).cuda()
                c = kept.numel()
                for pool in (k, v):
                    pool[to[0][:c], to[1][:c], a] = pool[page[kept], slot[kept], a]
                mass[to[0][:c], a, to[1][:c]] = mass[page[kept], a, slot[kept]]
        return {"k": k, "v": v, "mass": mass, "kept": None, "new_len": None}
    out = torch.zeros((n, h, case["heads"] // h, d), dtype=torch.float64, device="cuda")
    mass = s["mass"].double() if s["mass"] is not None else None
    for i, length in enumerate(s["len"].tolist()):
        where = _rows(s, i, length)
        if not where:
            continue
        q = s["q"][i].double().view(h, -1, d)
        for a in range(h):
            k, v = s["k"][where[0], where[1], a].double(), s["v"][where[0], where[1], a].double()
            p = torch.softmax(q[a] @ k.T / math.sqrt(d), -1)
            out[i, a] = p @ v
            if mass is not None:
                mass[where[0], a, where[1]] += p.sum(0)
    out = out.view(n, -1)
    return {"out": out} if mass is None else {"out": out, "mass": mass}
