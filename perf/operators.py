"""Operators of the paged KV cache of the gated full-attention layers, as measured.

Four operators that a serving step of the draft-tree cycle runs around its
tree-masked attention verify:

  plan    block tables grown and shrunk from request lengths, and the maps made
          of them: query offsets, key offsets, the key slots of every request,
          the slots and positions of the new tokens
  append  the K / V rows of new tokens written to their cache slots
  attend  causal attention of a chunk of new tokens (one token to a whole
          prompt) over the paged cache, grouped heads, packed requests
  commit  the K / V rows of the accepted tree path moved to consecutive
          positions after a verify

`run` computes them in plain torch operations in 32 bits, or, where `own` is
set, by the calls that a user of dforktree_b200 makes.
"""
import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------ cases --
def listed():
    att = dict(op="attend", Hq=16, Hkv=4, D=256, dtype="bf16", page=16)
    plan = dict(op="plan", page=16)
    app = dict(op="append", Hq=16, Hkv=4, D=256, dtype="bf16")
    com = dict(op="commit", Hkv=4, D=256, N=32, P=24, dtype="bf16", page=16)
    return [
        # one user's next token: a short conversation, latency only
        dict(att, name="attend one token", B=1, fresh=1, cached=700, lens="even"),
        # a full decode batch at the cycle's prefix length
        dict(att, name="attend decode batch", B=64, fresh=1, cached=4096, lens="ragged"),
        # a long document read in a serving step's chunk, tokens spread over single-token pages
        dict(att, name="attend long chunk", B=1, fresh=512, cached=32768, lens="even", page=1),
        # a whole prompt from an empty cache
        dict(att, name="attend whole prompt", B=1, fresh=8192, cached=0, lens="even"),
        # prompts of different lengths packed into one call; half precision, the narrower head
        dict(att, name="attend packed prompts", B=12, fresh=1100, cached=0, lens="ragged", Hq=16, Hkv=8, D=128,
             dtype="f16", page=64),
        # chunked prefill beside decodes: most requests bring one token, some a chunk
        dict(att, name="attend mixed batch", B=24, fresh=250, cached=3000, lens="mixed", Hq=16, Hkv=2, D=128),
        # a verify step of a small batch: 32 tree nodes in, the rejected ones' pages back
        dict(plan, name="plan small step", B=4, fresh=32, cached=500, keep=5, lens="ragged"),
        # the same for a large batch with long contexts
        dict(plan, name="plan large step", B=512, fresh=32, cached=8192, keep=5, lens="ragged"),
        # new tokens of a decode batch
        dict(app, name="append decode batch", B=64, fresh=1, lens="even"),
        # a step's worth of prompt tokens
        dict(app, name="append prompts", B=16, fresh=1000, lens="ragged"),
        # accepted paths of a small batch, the attention layers of an eighth of the model
        dict(com, name="commit small batch", B=2, layers=1, cached=300),
        # the cycle's batch over eight attention layers
        dict(com, name="commit full batch", B=64, layers=8, cached=1000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "attend", "plan", "append", "commit"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    page = rng.choice([1, 4, 16, 64])
    Hkv, D = rng.choice([(4, 256), (2, 256), (8, 128), (2, 128), (4, 64)])
    if op == "attend":
        G = rng.choice([1, 2, 3, 4, 8])
        while True:
            lens = rng.choice(["even", "ragged", "mixed"])
            B = _log(rng, 1, 64)
            fresh = rng.choice([1, _log(rng, 1, 8192), _log(rng, 2, 1024)])
            cached = rng.choice([0, _log(rng, 1, 32768)])
            case = dict(op=op, B=B, fresh=fresh, cached=cached, lens=lens, Hq=G * Hkv, Hkv=Hkv, D=D, dtype=dtype,
                        page=page)
            # no dearer than the whole prompt above, and its plain form's scores and keys fit
            if (4 * B * G * Hkv * fresh * (fresh + cached) <= 4 * 16 * 8192 * 8192
                    and B * (fresh + cached) * Hkv * D <= 64 * 4200 * 4 * 256
                    and work(case)["flops"] <= work(listed()[3])["flops"]):
                return case
    if op == "plan":
        B = _log(rng, 1, 512)
        return dict(op=op, B=B, fresh=rng.choice([1, 16, 32, 64, _log(rng, 1, 2000)]), cached=_log(rng, 1, 6000),
                    keep=rng.randint(0, 24), lens=rng.choice(["even", "ragged"]), page=page)
    if op == "append":
        return dict(op=op, B=_log(rng, 1, 64), fresh=_log(rng, 1, 250), Hq=4 * Hkv, Hkv=Hkv, D=D, dtype=dtype,
                    lens=rng.choice(["even", "ragged"]))
    return dict(op=op, B=_log(rng, 1, 64), layers=rng.randint(1, 8), Hkv=Hkv, D=D, N=rng.choice([16, 32, 64]),
                P=rng.randint(2, 24), cached=_log(rng, 1, 1000), dtype=dtype, page=page)


# ------------------------------------------------- lengths of the requests --
def _rng(case, salt):
    return random.Random(sum(v * w for v, w in zip((case["B"], case.get("fresh", 0), case.get("cached", 0), salt),
                                                   (1, 101, 10007, 1000003))))


def _spread(case, key, salt, low):
    """One length per request, up to case[key]: a fixed function of the case."""
    B, top, r = case["B"], case[key], _rng(case, salt)
    if case["lens"] == "even" or B == 1:
        return [top] * B
    return [max(min(low, top), int(top * r.uniform(0.3, 1.0))) for _ in range(B)]


def _lens(case):
    """(tokens already cached, new tokens) of each request."""
    cached, fresh = _spread(case, "cached", 1, 0), _spread(case, "fresh", 2, 1)
    if case["lens"] == "mixed":
        fresh = [f if b % 6 == 3 else 1 for b, f in enumerate(fresh)]
    return cached, fresh


def _cum(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def _i32(v, dev="cuda"):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _i64(v, dev="cuda"):
    return torch.tensor(v, dtype=torch.int64, device=dev)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _slots(lens, page, gen, spare):
    """Random pages for requests of these lengths: (key offsets, key slots, slots in the cache)."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    perm = torch.randperm(pages, device="cuda", generator=gen)
    n, off, first = _i64(lens), _i64(_cum(lens)), _i64(_cum(need))
    b = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), n)
    j = torch.arange(int(off[-1]), device="cuda") - off[b]
    return off.to(torch.int32), (perm[first[b] + j // page] * page + j % page).to(torch.int32), pages * page


# ---------------------------------------------------------------- prepare --
def prepare(case, seed):
    return {"attend": _prepare_attend, "plan": _prepare_plan, "append": _prepare_append,
            "commit": _prepare_commit}[case["op"]](case, _gen(seed))


def _randn(gen, dtype, *shape):
    return torch.randn(*shape, device="cuda", generator=gen, dtype=_DT[dtype])


def _prepare_attend(case, g):
    cached, fresh = _lens(case)
    total = [c + f for c, f in zip(cached, fresh)]
    kv_indptr, kv_indices, slots = _slots(total, case["page"], g, 5)
    return dict(op="attend", q=_randn(g, case["dtype"], sum(fresh), case["Hq"], case["D"]),
                k=_randn(g, case["dtype"], slots, case["Hkv"], case["D"]),
                v=_randn(g, case["dtype"], slots, case["Hkv"], case["D"]),
                qo_indptr=_i32(_cum(fresh)), kv_indptr=kv_indptr, kv_indices=kv_indices,
                nmax=max(fresh), lmax=max(total), scale=case["D"] ** -0.5)


def _prepare_plan(case, g):
    cached, fresh = _lens(case)
    B, page = case["B"], case["page"]
    held = [-(-c // page) for c in cached]
    grown = [-(-(c + f) // page) for c, f in zip(cached, fresh)]
    n_pages, rows, width = sum(grown) + 7, B + 3, max(grown) + 2
    perm = torch.randperm(n_pages, device="cuda", generator=g)
    row = torch.randperm(rows, device="cuda", generator=g)[:B]
    # each request's pages come off the end of the permutation; the rest is the free stack
    n, first = _i64(held), _i64(_cum(held))
    b = torch.repeat_interleave(torch.arange(B, device="cuda"), n)
    j = torch.arange(sum(held), device="cuda")
    table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    table[row[b], j - first[b]] = perm[n_pages - 1 - j].to(torch.int32)
    held_rows = torch.zeros(rows, dtype=torch.int32, device="cuda")
    held_rows[row] = n.to(torch.int32)
    keep = torch.minimum(torch.randint(0, case["keep"] + 1, (B,), device="cuda", generator=g), _i64(fresh))

    def outputs(tokens, keys):
        return dict(qo_indptr=torch.zeros(B + 1, dtype=torch.int32, device="cuda"),
                    kv_indptr=torch.zeros(B + 1, dtype=torch.int32, device="cuda"),
                    kv_indices=torch.zeros(keys, dtype=torch.int32, device="cuda"),
                    slot_map=torch.zeros(tokens, dtype=torch.int64, device="cuda"),
                    positions=torch.zeros(tokens, dtype=torch.int64, device="cuda"))
    keys = sum(cached) + sum(fresh)
    # the new tokens' buffers are padded, as a captured step keeps them
    return dict(op="plan", page=page, rows=row, cached=_i64(cached), fresh=_i64(fresh), none=_i64([0] * B),
                kept=_i64(cached) + keep, table=table, held=held_rows, free=perm.to(torch.int32),
                n_free=_i32([n_pages - sum(held)]), grow=outputs(sum(fresh) + 9, keys), trim=outputs(1, keys))


def _prepare_append(case, g):
    _, fresh = _lens(dict(case, cached=0))
    T, Hq, Hkv, D = sum(fresh), case["Hq"], case["Hkv"], case["D"]
    slots = T + 64
    # K and V are slices of the layer's fused projection
    qkv = _randn(g, case["dtype"], T, (Hq + 2 * Hkv) * D)
    k = qkv[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)
    v = qkv[:, (Hq + Hkv) * D:].view(T, Hkv, D)
    slot = torch.randperm(slots, device="cuda", generator=g)[:T]
    slot = torch.where(torch.arange(T, device="cuda") % 97 == 96, -1, slot)       # padding rows of a captured step
    return dict(op="append", k=k, v=v, kc=_randn(g, case["dtype"], slots, Hkv, D),
                vc=_randn(g, case["dtype"], slots, Hkv, D), slot=slot)


def _prepare_commit(case, g):
    B, N, P = case["B"], case["N"], case["P"]
    r = _rng(case, 3)
    lens = [N + r.randint(0, case["cached"]) for _ in range(B)]
    kv_indptr, kv_indices, slots = _slots(lens, case["page"], g, 5)
    # the accepted path: the root, then ascending node ids
    alen = torch.randint(1, min(N, P) + 1, (B,), device="cuda", generator=g)
    pick = torch.rand(B, N, device="cuda", generator=g)
    pick[:, 0] = -1.0
    path = pick.argsort(1)[:, :P]
    past = torch.arange(min(N, P), device="cuda")[None] >= alen[:, None]
    path = torch.where(past, N, path).sort(1).values
    path = torch.where(path == N, -1, path)
    path = torch.cat([path, path.new_full((B, P - path.shape[1]), -1)], 1)
    return dict(op="commit", N=N, kv_indptr=kv_indptr, kv_indices=kv_indices, path=path, alen=alen,
                kc=_randn(g, case["dtype"], case["layers"], slots, case["Hkv"], case["D"]),
                vc=_randn(g, case["dtype"], case["layers"], slots, case["Hkv"], case["D"]))


# -------------------------------------------------------------------- run --
def run(state):
    if own:
        return _OWN[state["op"]](state)
    return _PLAIN[state["op"]](state)


def _own_attend(s):
    from dforktree_b200 import kernels as K
    return K.chunk_attention(s["q"], s["k"], s["v"], s["qo_indptr"], s["kv_indptr"], s["kv_indices"],
                             sm_scale=s["scale"])


def _own_plan(s):
    from dforktree_b200 import kernels as K
    # grow by the tree's nodes for the verify, then give back what the rejected ones took
    K.page_plan(s["cached"], s["fresh"], s["table"], s["held"], s["free"], s["n_free"], s["page"], rows=s["rows"],
                out=s["grow"])
    K.page_plan(s["kept"], s["none"], s["table"], s["held"], s["free"], s["n_free"], s["page"], rows=s["rows"],
                out=s["trim"])
    return _plan_outputs(s)


def _own_append(s):
    from dforktree_b200 import kernels as K
    K.kv_append(s["k"], s["v"], s["kc"], s["vc"], s["slot"])
    return s["kc"], s["vc"]


def _own_commit(s):
    from dforktree_b200 import kernels as K
    K.kv_commit(s["kc"], s["vc"], s["kv_indptr"], s["kv_indices"], s["path"], s["alen"], s["N"])
    return s["kc"], s["vc"]


def _plan_outputs(s):
    return dict(grow=s["grow"], trim=s["trim"], table=s["table"], held=s["held"], free=s["free"], n_free=s["n_free"])


def _plain_attend(s):
    q, k, v = s["q"], s["k"], s["v"]
    T, Hq, D = q.shape
    Hkv, nmax, lmax = k.shape[1], s["nmax"], s["lmax"]
    qo, kv = s["qo_indptr"].long(), s["kv_indptr"].long()
    B, G = qo.numel() - 1, Hq // Hkv
    n, length = qo[1:] - qo[:-1], kv[1:] - kv[:-1]
    i, j = torch.arange(nmax, device=q.device), torch.arange(lmax, device=q.device)
    # keys and queries of every request, padded to the longest
    at = s["kv_indices"][(kv[:-1, None] + j).clamp(max=s["kv_indices"].numel() - 1)].long()       # [B, lmax]
    row = (qo[:-1, None] + i).clamp(max=T - 1)                                                    # [B, nmax]
    kf = k[at].float().permute(0, 2, 3, 1)                                                        # [B, Hkv, D, lmax]
    vf = v[at].float().permute(0, 2, 1, 3)                                                        # [B, Hkv, lmax, D]
    qf = q[row].float().view(B, nmax, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * nmax, D)
    score = (qf @ kf).view(B, Hkv, G, nmax, lmax) * s["scale"]
    # token i of a request's n new ones sees its keys up to length - n + i
    seen = (j <= (length - n)[:, None, None] + i[:, None]) & (j < length[:, None, None])          # [B, nmax, lmax]
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
    total = e.sum(-1, keepdim=True)
    o = (e.view(B, Hkv, G * nmax, lmax) @ vf).view(B, Hkv, G, nmax, D) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(B * nmax, Hq, D)
    # row t of the packed output
    t = torch.arange(T, device=q.device)
    b = torch.searchsorted(qo[1:], t, right=True)
    return o[b * nmax + t - qo[b]].to(q.dtype)


def _plain_plan_one(s, cached, fresh, out):
    """Requests in order give back the pages past their new length, then take
    new ones off the top of the free stack."""
    page, rows, table, held, free, n_free = s["page"], s["rows"], s["table"], s["held"], s["free"], s["n_free"]
    dev, n_pages = table.device, free.numel()
    have, length = held[rows].long(), cached + fresh
    need = (length + page - 1) // page
    back, take = (have - need).clamp(min=0), (need - have).clamp(min=0)
    p = torch.arange(table.shape[1], device=dev)
    old = table[rows].long()
    stack = torch.cat([free.long(), free.new_zeros(1).long()])
    gone = (p >= need[:, None]) & (p < have[:, None])
    at = n_free + (back.cumsum(0) - back)[:, None] + p - need[:, None]
    stack.scatter_(0, torch.where(gone, at, n_pages).flatten(), old.flatten())
    top = n_free + back.sum()
    come = (p >= have[:, None]) & (p < need[:, None])
    at = top - 1 - ((take.cumsum(0) - take)[:, None] + p - have[:, None])
    new = torch.where(come, stack[torch.where(come, at, 0)], old)
    table[rows] = new.to(torch.int32)
    held[rows] = need.to(torch.int32)
    free.copy_(stack[:-1])
    n_free.copy_(top - take.sum())
    qo, kv = torch.nn.functional.pad(fresh.cumsum(0), (1, 0)), torch.nn.functional.pad(length.cumsum(0), (1, 0))
    out["qo_indptr"].copy_(qo)
    out["kv_indptr"].copy_(kv)
    B = rows.numel()
    j = torch.arange(out["kv_indices"].numel(), device=dev)
    b = torch.searchsorted(kv[1:], j, right=True).clamp(max=B - 1)
    off = torch.where(j < kv[-1], j - kv[b], 0)
    out["kv_indices"].copy_(torch.where(j < kv[-1], new[b, off // page] * page + off % page, out["kv_indices"]))
    t = torch.arange(out["slot_map"].numel(), device=dev)
    b = torch.searchsorted(qo[1:], t, right=True).clamp(max=B - 1)
    off = torch.where(t < qo[-1], cached[b] + t - qo[b], 0)
    out["slot_map"].copy_(torch.where(t < qo[-1], new[b, off // page] * page + off % page, -1))
    out["positions"].copy_(off)


def _plain_plan(s):
    _plain_plan_one(s, s["cached"], s["fresh"], s["grow"])
    _plain_plan_one(s, s["kept"], s["none"], s["trim"])
    return _plan_outputs(s)


def _plain_append(s):
    # a padding row writes nothing: its target takes what it holds
    k, v, kc, vc, slot = s["k"], s["v"], s["kc"], s["vc"], s["slot"]
    live = torch.nonzero(slot >= 0)[:, 0]
    kc[slot[live]] = k[live]
    vc[slot[live]] = v[live]
    return kc, vc


def _plain_commit(s):
    kc, vc, path, alen, N = s["kc"], s["vc"], s["path"], s["alen"], s["N"]
    first = s["kv_indptr"][1:].long() - N                                     # the tree's first key of each request
    i = torch.arange(path.shape[1], device=path.device)
    b, i = torch.nonzero((i < alen[:, None]) & (path >= 0), as_tuple=True)
    to, src = s["kv_indices"][first[b] + i].long(), s["kv_indices"][first[b] + path[b, i]].long()
    kc[:, to] = kc[:, src]
    vc[:, to] = vc[:, src]
    return kc, vc


_OWN = {"attend": _own_attend, "plan": _own_plan, "append": _own_append, "commit": _own_commit}
_PLAIN = {"attend": _plain_attend, "plan": _plain_plan, "append": _plain_append, "commit": _plain_commit}


# ------------------------------------------------------------------- work --
def work(case):
    if case["op"] == "attend":
        cached, fresh = _lens(case)
        pairs = sum(f * c + f * (f + 1) // 2 for c, f in zip(cached, fresh))
        keys, T = sum(cached) + sum(fresh), sum(fresh)
        return {"bytes": 2 * T * case["Hq"] * case["D"] * 2 + keys * (2 * case["Hkv"] * case["D"] * 2 + 4),
                "flops": 4 * pairs * case["Hq"] * case["D"]}
    if case["op"] == "plan":
        cached, fresh = _lens(case)
        page = case["page"]
        keys, T = sum(cached) + sum(fresh), sum(fresh)
        # pages read and slots written by both calls, the new tokens' slots and positions, lengths and offsets
        return {"bytes": 4 * (2 * keys + 2 * (keys // page)) + 16 * T + 2 * case["B"] * (8 * 3 + 4 * 4), "flops": 0}
    if case["op"] == "append":
        T = sum(_lens(dict(case, cached=0))[1])
        return {"bytes": T * (8 + 2 * 2 * case["Hkv"] * case["D"] * 2), "flops": 0}
    # half of the path's longest, on average, moves: read once, written once
    moved = case["B"] * case["layers"] * (min(case["N"], case["P"]) // 2)
    return {"bytes": 2 * 2 * moved * case["Hkv"] * case["D"] * 2 + 8 * case["B"] * case["P"], "flops": 0}


# ------------------------------------------------------------------ exact --
def exact(case, seed):
    """The operators by their definition, request by request, in 64 bits."""
    s = prepare(case, seed)
    if s["op"] != "attend":
        return None if s["op"] == "plan" else _exact_move(s)
    T, Hq, D = s["q"].shape
    Hkv = s["k"].shape[1]
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device="cuda")
    qo, kv = s["qo_indptr"].tolist(), s["kv_indptr"].tolist()
    for b in range(len(qo) - 1):
        slot = s["kv_indices"][kv[b]:kv[b + 1]].long()
        n, length = qo[b + 1] - qo[b], kv[b + 1] - kv[b]
        last = torch.arange(n, device="cuda") + (length - n)
        for h in range(Hq):
            q = s["q"][qo[b]:qo[b + 1], h].double()
            k, v = s["k"][slot, h // (Hq // Hkv)].double(), s["v"][slot, h // (Hq // Hkv)].double()
            w = torch.mm(q, k.t()).mul_(s["scale"])
            w.masked_fill_(torch.arange(length, device="cuda")[None, :] > last[:, None], float("-inf"))
            out[qo[b]:qo[b + 1], h] = torch.mm(torch.softmax(w, 1), v)
    return out


def _exact_move(s):
    kc, vc = s["kc"].double(), s["vc"].double()
    if s["op"] == "append":
        for t, to in enumerate(s["slot"].tolist()):
            if to >= 0:
                kc[to], vc[to] = s["k"][t].double(), s["v"][t].double()
        return kc, vc
    end, path, alen = s["kv_indptr"].tolist(), s["path"].tolist(), s["alen"].tolist()
    for b, n in enumerate(alen):
        tree = s["kv_indices"][end[b + 1] - s["N"]:end[b + 1]].tolist()
        for i in range(n):
            if path[b][i] >= 0:
                kc[:, tree[i]] = s["kc"][:, tree[path[b][i]]].double()
                vc[:, tree[i]] = s["vc"][:, tree[path[b][i]]].double()
    return kc, vc
