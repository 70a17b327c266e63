"""Workloads of the operators on the int8 KV cache: attention of a tree of
drafted tokens, the commit of its accepted path, and a cache that evicts by
accumulated attention weight.

The cache is the library's: per sequence K int8 [slot][kv_heads * head_dim]
with one f32 scale per slot, V int8 slot-interleaved
[(slot / 4)][kv_heads * head_dim][slot % 4] with one f32 scale per slot.  A
query head is quantised to int8 with one scale, so q . k is a whole number.

Kinds of case ("op"):
  tree    attend_tree_q8: T nodes per sequence attend to the committed slots
          and to their ancestors (mask words) or, without a mask, to the
          nodes before them
  accum   attend_accum_q8: the weights of the taken nodes added to the slots'
          accumulated weight
  decode  attend_acc_q8: one token per sequence, attention and accumulation
  accept  tree_verify + kv_accept: the accepted path of the tree, its rows
          moved behind the committed ones in every layer
  evict   kv_evict_q8: the budget's slots kept, their rows moved into the
          evicted slots

Each case runs in a plain form (elementary torch operations in 32 bits) or,
where ``own`` is true, through fastgemma_b200.device.
"""
import math

import numpy as np
import torch

own = False


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the smallest step: a chain of four drafts over a short prompt, one sequence
        dict(name="tree_chain4", op="tree", B=1, T=4, len=96, heads=8, kvh=2, hd=256, shape="chain",
             window=0, ragged=0),
        # a batch of eight at the decode step's context of 1024, 16-node trees,
        # a sliding-window layer whose cache is a ring
        dict(name="tree_ring_8x16", op="tree", B=8, T=16, len=1024, heads=8, kvh=2, hd=256,
             shape="tree", window=512, ragged=1),
        # a full-attention layer, longer contexts of different lengths, 61-node trees
        dict(name="tree_4x61_8k", op="tree", B=4, T=61, len=8191, heads=8, kvh=2, hd=256,
             shape="tree", window=0, ragged=1),
        # a whole prefill chunk of 256 tokens behind a 16K context
        dict(name="chunk_256_16k", op="tree", B=1, T=256, len=16384, heads=8, kvh=2, hd=256,
             shape="chain", window=0, ragged=0),
        # the weights of accepted 16-node paths over eight contexts
        dict(name="accum_8x16_4k", op="accum", B=8, T=16, len=4096, heads=8, kvh=2, hd=256,
             shape="tree", window=0, ragged=1),
        # a prefill chunk's weights over a 16K context
        dict(name="accum_256_16k", op="accum", B=1, T=256, len=16384, heads=8, kvh=2, hd=256,
             shape="chain", window=0, ragged=0),
        # one sequence decoding at an odd length
        dict(name="decode_1x1000", op="decode", B=1, len=1001, heads=8, kvh=2, hd=256, ragged=0),
        # eight sequences decoding over long caches of different lengths
        dict(name="decode_8x32k", op="decode", B=8, len=32768, heads=8, kvh=2, hd=256, ragged=1),
        # one sequence, six drafts, four layers
        dict(name="accept_1x6", op="accept", B=1, T=6, L=4, len=500, kvh=2, hd=256, ragged=0),
        # the decode stack's 30 layers, eight sequences, 61-node trees
        dict(name="accept_8x61", op="accept", B=8, T=61, L=30, len=1024, kvh=2, hd=256, ragged=1),
        # one short cache back to its budget
        dict(name="evict_1x600", op="evict", B=1, len=600, budget=512, sink=4, recent=64, kvh=2,
             hd=256, ragged=0),
        # eight long caches back to 7/8 of their slots
        dict(name="evict_8x16k", op="evict", B=8, len=16384, budget=14336, sink=4, recent=256,
             kvh=2, hd=256, ragged=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "accum", "decode", "decode", "accept", "evict"])
    kvh, grp, hd = rng.choice([1, 2, 2, 4]), rng.choice([1, 2, 4, 4, 8]), rng.choice(
        [64, 128, 192, 256, 256, 512])
    c = dict(op=op, B=_log(rng, 1, 16), len=_log(rng, 1, 20000), kvh=kvh, hd=hd,
             ragged=rng.randint(0, 1))
    if op in ("tree", "accum"):
        c.update(T=_log(rng, 1, 256), heads=kvh * grp, shape=rng.choice(["chain", "tree"]),
                 window=rng.choice([0, 0, _log(rng, 16, 2048)]))
        most = 256 * 16640 * 8 * 256
        cost = lambda: c["B"] * c["T"] * (c["len"] + c["T"]) * c["heads"] * hd  # noqa: E731
    elif op == "decode":
        c.update(heads=kvh * grp)
        most = 8 * 24576 * 2 * 256
        cost = lambda: c["B"] * c["len"] * kvh * hd  # noqa: E731
    elif op == "accept":
        c.update(T=_log(rng, 1, 256), L=_log(rng, 1, 30), len=min(c["len"], 2000))
        most = 8 * 61 * 30 * 512
        cost = lambda: c["B"] * c["T"] * c["L"] * kvh * hd  # noqa: E731
    else:
        c["len"] = max(8, c["len"])
        keep = max(1, int(c["len"] * rng.uniform(0.5, 1.0)))
        c.update(budget=keep, sink=min(keep // 4, 4), recent=keep // rng.randint(2, 16))
        most = 8 * 16384 * 512
        cost = lambda: c["B"] * c["len"] * kvh * hd  # noqa: E731
    while cost() > most:
        k = "B" if c["B"] > 1 else ("L" if c.get("L", 1) > 1 else "T" if c.get("T", 1) > 32 else "len")
        c[k] = max(1, c[k] * 2 // 3)
    if op == "evict":
        c["budget"] = min(c["budget"], c["len"])
    return c


def _lens(c):
    """Committed lengths: all `len`, or spread down to half of it."""
    n, B = c["len"], c["B"]
    return [n - (n * b // (2 * B) if c["ragged"] else 0) for b in range(B)]


def _nodes(c):
    return c.get("T", 1 if c["op"] == "decode" else 0)


def _ring(c):
    """A sliding-window layer's ring: the window and the nodes, in whole groups of 16."""
    w = c.get("window", 0)
    return (w + c["T"] + 15) // 16 * 16 if w else 0


def _cap(c):
    return _ring(c) or (c["len"] + _nodes(c) + 15) // 16 * 16


def work(c):
    kvd = c["kvh"] * c["hd"]
    if c["op"] in ("tree", "accum", "decode"):
        T, H, hd = _nodes(c), c["heads"], c["hd"]
        w = c.get("window", 0)
        n = [min(x, w) if w else x for x in _lens(c)]
        slots = sum(n) + c["B"] * T
        # visible (query, slot) pairs: a window's width, else the committed slots; half the nodes
        pairs = T * (sum(n) + c["B"] * (T + 1) / 2)
        rows = c["B"] * T
        mask = rows * ((T + 63) // 64) * 8 if c.get("shape") == "tree" else 0
        if c["op"] == "accum":
            return {"bytes": slots * (kvd + 4 + 8) + rows * H * (hd * 4 + 4) + mask,
                    "flops": 2 * pairs * H * hd}
        acc = slots * 8 if c["op"] == "decode" else rows * H * 4
        return {"bytes": slots * (2 * kvd + 8) + rows * H * hd * 8 + mask + acc,
                "flops": 4 * pairs * H * hd}
    if c["op"] == "accept":
        # the tree's words, and half of a path of about log2(T) + 1 nodes moved
        moved = c["B"] * c["L"] * (math.log2(c["T"]) + 1) / 2
        return {"bytes": c["B"] * c["T"] * 16 + moved * 2 * (2 * kvd + 8), "flops": 0}
    n = sum(_lens(c))
    moved = 0.0
    for x in _lens(c):
        gone = max(0, x - c["budget"])
        movable = max(1, x - c["sink"] - c["recent"])
        moved += min(gone, gone * max(0, c["budget"] - c["sink"]) / movable)
    return {"bytes": n * 8 + c["B"] * c["budget"] * 12 + moved * 2 * (2 * kvd + 8), "flops": 0}


# ------------------------------------------------------------------ inputs
def _cache(c, gen, layers=0):
    """Rows as the projections leave them (N(0, 1), one scale per row); what
    no token has written yet holds any bytes and scales that are no numbers."""
    B, kvd, cap = c["B"], c["kvh"] * c["hd"], _cap(c)
    lead = (layers, B) if layers else (B,)
    used = min(cap, c["len"] + _nodes(c))

    def rows(n):
        x = torch.randn(lead + (n, kvd), device="cuda", generator=gen)
        s = x.abs().amax(-1) / 127.0
        return torch.round(x / s[..., None]).to(torch.int8), s

    kc = torch.full(lead + (cap, kvd), 77, dtype=torch.int8, device="cuda")
    vt = torch.full(lead + (cap // 4, kvd, 4), -99, dtype=torch.int8, device="cuda")
    ks, vs = (torch.full(lead + (cap,), math.nan, device="cuda") for _ in range(2))
    kc[..., :used, :], ks[..., :used] = rows(used)
    v, vs[..., :used] = rows(used)
    pad = torch.nn.functional.pad(v, (0, 0, 0, -used % 4), value=-99)
    vt[..., : pad.shape[-2] // 4, :, :] = pad.unflatten(-2, (-1, 4)).transpose(-1, -2)
    if not _ring(c):  # shorter sequences end earlier
        late = torch.arange(cap, device="cuda")[None] >= (
            torch.tensor(_lens(c), device="cuda") + _nodes(c))[:, None]
        ks.masked_fill_(late, math.nan)
        vs.masked_fill_(late, math.nan)
    return kc, ks, vt, vs


def _trees(c, gen):
    """Random trees: each node hangs under one of the four before it (or is a chain)."""
    B, T = c["B"], c["T"]
    back = torch.randint(1, 5, (B, T), device="cuda", generator=gen)
    i = torch.arange(T, device="cuda")[None]
    parent = (i - (back if c.get("shape", "tree") == "tree" else 1)).clamp(min=0)
    parent = torch.where(i == 0, -1, parent).to(torch.int32)
    up = parent.cpu().numpy()
    see, depth = np.zeros((B, T, T), bool), np.zeros((B, T), np.int64)
    rows = np.arange(B)
    for n in range(T):
        if n:
            see[:, n] = see[rows, up[:, n]]
            depth[:, n] = depth[rows, up[:, n]] + 1
        see[:, n, n] = True
    return parent, torch.from_numpy(see).cuda(), torch.from_numpy(depth).cuda()


def _words(see):
    """Bool [B][T][T] -> mask words [B][T][ceil(T / 64)], bit j % 64 of word j / 64."""
    bits = np.packbits(see.cpu().numpy(), axis=-1, bitorder="little")
    bits = np.pad(bits, ((0, 0), (0, 0), (0, -bits.shape[-1] % 8)))
    return torch.from_numpy(np.ascontiguousarray(bits).view(np.int64)).cuda()


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, T = c["B"], _nodes(c)
    s = {"c": c, "lens": torch.tensor(_lens(c), dtype=torch.int32, device="cuda")}
    s["kc"], s["ks"], s["vt"], s["vs"] = _cache(c, gen, c.get("L", 0))
    if c["op"] in ("tree", "accum", "decode"):
        H, hd = c["heads"], c["hd"]
        # normalised query heads under norm weights that give scores of a few units
        s["q"] = torch.randn(B * T, H * hd, device="cuda", generator=gen) * (4.0 / math.sqrt(hd))
    if c["op"] in ("tree", "accum"):
        _, see, depth = _trees(c, gen)
        s["see"] = see
        s["mask"] = _words(see) if c["shape"] == "tree" else None
        s["pos"] = (s["lens"][:, None] + depth).to(torch.int32).reshape(-1)
    if c["op"] in ("accum", "decode"):
        s["acc"] = torch.rand(B, _cap(c), device="cuda", generator=gen)
    if c["op"] == "accum":
        s["take"] = (torch.rand(B, T, device="cuda", generator=gen) < 0.5).to(torch.uint8)
        s["lse"] = _plain_attend(s, True)[1]
    if c["op"] == "accept":
        parent, see, _ = _trees(c, gen)
        token = torch.randint(0, 2, (B, T), device="cuda", generator=gen, dtype=torch.int32)
        target = torch.randint(0, 2, (B, T), device="cuda", generator=gen, dtype=torch.int32)
        s.update(parent=parent, see=see, token=token, target=target)
    if c["op"] == "evict":
        cap = _cap(c)
        s["acc"] = torch.rand(B, cap, device="cuda", generator=gen) ** 8 * 10
        # a few slots with equal weights
        s["acc"] = torch.where(s["acc"] < 1e-9, 0.0, s["acc"])
        s["tpos"] = torch.arange(cap, device="cuda", dtype=torch.int32).repeat(B, 1)
        s["acc_out"] = torch.zeros(B, c["budget"], device="cuda")
        s["tpos_out"] = torch.zeros(B, c["budget"], dtype=torch.int32, device="cuda")
        s["map"] = torch.zeros(B, c["budget"], dtype=torch.int32, device="cuda")
        s["lens_out"] = torch.zeros(B, dtype=torch.int32, device="cuda")
    if own:
        _handles(s)
    torch.cuda.synchronize()
    return s


def _handles(s):
    """The views, outputs and workspaces that a program keeps from step to step."""
    from fastgemma_b200 import device as D
    c = s["c"]
    views = [D.KvCache(*(s[k][l] for k in ("kc", "ks", "vt", "vs")), c["kvh"], c["hd"])
             for l in range(c["L"])] if "L" in c else None
    if views:
        B, T = c["B"], c["T"]
        s["kv"] = D.kv_layers(views)
        s["path"] = torch.empty(B, T, dtype=torch.int32, device="cuda")
        s["n_acc"], s["next"], s["lens_new"] = (
            torch.empty(B, dtype=torch.int32, device="cuda") for _ in range(3))
        return
    s["kv"] = D.KvCache(s["kc"], s["ks"], s["vt"], s["vs"], c["kvh"], c["hd"], ring=_ring(c),
                        acc=s.get("acc"), tpos=s.get("tpos"))
    if c["op"] in ("tree", "accum", "decode"):
        s["out"] = torch.empty_like(s["q"])
        s["lse_out"] = torch.empty(s["q"].shape[0], c["heads"], device="cuda")
        s["ws"] = D.attend_workspace(s["kv"], c["heads"], _nodes(c))


# ------------------------------------------------------------- plain forms
def _visible(s):
    """Bool [B][T][slot]: what each node sees.  In a ring, slot x holds the
    newest position that is x modulo the ring."""
    c = s["c"]
    T, cap, ring, w = _nodes(c), _cap(c), _ring(c), c.get("window", 0)
    lens = s["lens"].long()[:, None]
    x = torch.arange(cap, device="cuda")[None]
    t = lens + T - 1 - (lens + T - 1 - x) % ring if ring else x.expand(len(lens), cap)
    node = (t - lens).clamp(0, T - 1)
    see = s["see"] if "see" in s else torch.ones(c["B"], 1, 1, dtype=torch.bool, device="cuda")
    among = torch.gather(see, 2, node[:, None].expand(-1, T, -1))
    vis = torch.where((t < lens)[:, None], (t >= 0)[:, None], among & (t < lens + T)[:, None])
    if w:
        pos = s["pos"].reshape(c["B"], T).long()
        at = torch.where(t < lens, t, torch.gather(pos, 1, node))
        vis = vis & (at[:, None] > pos[..., None] - w)
    return vis


def _plain_scores(s):
    """Scores [B][kvh][group][T][slot] (whole-number dots times both scales), -inf where unseen."""
    c = s["c"]
    B, T, kvh, hd = c["B"], _nodes(c), c["kvh"], c["hd"]
    q = s["q"].reshape(B, T, kvh, -1, hd)
    top = q.abs().amax(-1, keepdim=True)
    inv = torch.where(top > 0, torch.full_like(top, 127.0) / top, 0.0)
    q8 = torch.round(q * inv).clamp(-127, 127)
    qs = top / torch.full_like(top, 127.0)
    k = s["kc"].float().unflatten(-1, (kvh, hd))
    dot = torch.einsum("btkgd,bnkd->bkgtn", q8, k)
    sc = dot * qs.permute(0, 2, 3, 1, 4) * s["ks"][:, None, None, None]
    return torch.where(_visible(s)[:, None, None], sc, -math.inf)


def _plain_attend(s, weights=False):
    c = s["c"]
    B, T, kvh, hd = c["B"], _nodes(c), c["kvh"], c["hd"]
    sc = _plain_scores(s)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m > -math.inf, m, 0.0))
    l = p.sum(-1, keepdim=True)
    lse = (m + torch.log(l)).squeeze(-1).permute(0, 3, 1, 2).reshape(B * T, -1)
    if weights:
        return p / l, lse
    v = s["vt"].transpose(-1, -2).flatten(1, 2).float().unflatten(-1, (kvh, hd))
    vs = torch.where(_visible(s).any(1), s["vs"], 0.0)
    o = torch.einsum("bkgtn,bnkd->btkgd", p * vs[:, None, None, None], v)
    o = o / l.permute(0, 3, 1, 2, 4)
    return o.reshape(B * T, -1), lse, p / l


def _plain_accum(s, weights, keep):
    """acc = keep * acc + weights; a slot that a node has just filled starts from 0."""
    lens, T, cap = s["lens"][:, None], _nodes(s["c"]), _cap(s["c"])
    x = torch.arange(cap, device="cuda")[None]
    old = torch.where(x < lens, keep * s["acc"], 0.0)
    s["acc"].copy_(torch.where(x < lens + T, old + weights, s["acc"]))
    return s["acc"]


DECAY = 0.96875


def _plain_accept(s):
    c = s["c"]
    T = c["T"]
    i = torch.arange(T, device="cuda")
    up = s["parent"].long().clamp(min=0)
    right = (s["token"] == torch.gather(s["target"], 1, up)) & (s["parent"] >= 0)
    # of right siblings the first counts
    twin = (up[:, :, None] == up[:, None, :]) & right[:, None, :] & (i[None, :] < i[:, None])[None]
    right = right & ~twin.any(-1)
    right[:, 0] = True
    taken = ~(s["see"] & ~right[:, None, :]).any(-1)
    path = torch.where(taken, i, T).sort(-1).values
    n = taken.sum(-1)
    last = torch.gather(path, 1, n[:, None] - 1)
    nxt = torch.gather(s["target"], 1, last)[:, 0]
    dst = s["lens"].long()[:, None] + i
    src = torch.where(path < T, s["lens"].long()[:, None] + path, dst)
    b = torch.arange(c["B"], device="cuda")[:, None]
    s["kc"][:, b, dst] = s["kc"][:, b, src]
    s["vt"][:, b, dst // 4, :, dst % 4] = s["vt"][:, b, src // 4, :, src % 4]
    s["ks"][:, b, dst] = s["ks"][:, b, src]
    s["vs"][:, b, dst] = s["vs"][:, b, src]
    return {"path": torch.where(path < T, path, -1).to(torch.int32), "n_acc": n.to(torch.int32),
            "next": nxt, "lens": (s["lens"] + n).to(torch.int32), **_state(s)}


def _plain_evict(s):
    c = s["c"]
    cap, budget = _cap(c), c["budget"]
    x = torch.arange(cap, device="cuda")[None]
    lens = s["lens"].long()[:, None]
    here = x < lens
    newest = torch.where(here, s["tpos"], -1).amax(-1, keepdim=True)
    safe = (s["tpos"] < c["sink"]) | (s["tpos"] > newest - c["recent"])
    key = torch.where(here, torch.where(safe, math.inf, s["acc"]), -math.inf)
    order = key.sort(stable=True, dim=-1, descending=True).indices
    rank = torch.empty_like(order).scatter_(1, order, x.expand_as(order).contiguous())
    keep = here & (rank < budget)
    late = torch.where(keep & (x >= budget), x, cap).sort(-1).values
    hole = (~keep[:, :budget]).cumsum(-1) - 1
    fill = torch.gather(late, 1, hole.clamp(min=0))
    y = x[:, :budget]
    new = torch.where(keep[:, :budget], y, torch.where(fill < cap, fill, -1))
    at = new.clamp(min=0)
    s["acc_out"].copy_(torch.where(new >= 0, torch.gather(s["acc"], 1, at), s["acc_out"]))
    s["tpos_out"].copy_(torch.where(new >= 0, torch.gather(s["tpos"], 1, at), s["tpos_out"]))
    b, dst = ((new != y) & (new >= 0)).nonzero(as_tuple=True)
    src = new[b, dst]
    s["kc"][b, dst] = s["kc"][b, src]
    s["vt"][b, dst // 4, :, dst % 4] = s["vt"][b, src // 4, :, src % 4]
    s["ks"][b, dst] = s["ks"][b, src]
    s["vs"][b, dst] = s["vs"][b, src]
    return {"map": new.to(torch.int32), "lens": lens[:, 0].clamp(max=budget).to(torch.int32),
            "acc": s["acc_out"], "tpos": s["tpos_out"], **_state(s)}


def _state(s):
    """The caches after a move: bytes and scales are moved, not computed, so they stay as they are."""
    return {k: s[k] for k in ("kc", "ks", "vt", "vs")}


def run(state):
    s, c = state, state["c"]
    if own:
        return _run_own(s, c)
    if c["op"] == "tree":
        out, lse, _ = _plain_attend(s)
        return {"out": out, "lse": lse}
    if c["op"] == "decode":
        out, _, p = _plain_attend(s)
        return {"out": out, "acc": _plain_accum(s, p.sum((1, 2, 3)), DECAY)}
    if c["op"] == "accum":
        lse = s["lse"].reshape(c["B"], -1, c["kvh"], c["heads"] // c["kvh"]).permute(0, 2, 3, 1)
        p = torch.exp(_plain_scores(s) - lse[..., None])
        p = p * s["take"][:, None, None, :, None]
        w = p.sum((1, 2, 3))
        if _ring(c):
            x = torch.arange(_cap(c), device="cuda")[None]
            end = s["lens"].long()[:, None] + c["T"] - 1
            t = end - (end - x) % _ring(c)
            old = torch.where(t < s["lens"][:, None], DECAY * s["acc"], 0.0)
            s["acc"].copy_(torch.where(t >= 0, old + w, s["acc"]))
            return {"acc": s["acc"]}
        return {"acc": _plain_accum(s, w, DECAY)}
    return _plain_accept(s) if c["op"] == "accept" else _plain_evict(s)


def _run_own(s, c):
    from fastgemma_b200 import device as D
    if c["op"] == "tree":
        D.attend_tree_q8(s["out"], s["q"], s["kv"], c["heads"], c["T"], s["lens"], mask=s["mask"],
                         pos=s["pos"], window=c["window"], lse=s["lse_out"], ws=s["ws"])
        return {"out": s["out"], "lse": s["lse_out"]}
    if c["op"] == "decode":
        D.attend_acc_q8(s["out"], s["q"], s["kv"], c["heads"], s["lens"], decay=DECAY, ws=s["ws"])
        return {"out": s["out"], "acc": s["acc"]}
    if c["op"] == "accum":
        D.attend_accum_q8(s["q"], s["kv"], c["heads"], c["T"], s["lens"], s["lse"], mask=s["mask"],
                          pos=s["pos"], window=c["window"], take=s["take"], decay=DECAY, ws=s["ws"])
        return {"acc": s["acc"]}
    if c["op"] == "accept":
        D.tree_verify(s["path"], s["n_acc"], s["next"], s["parent"], s["token"], s["target"])
        D.kv_accept(s["kv"], c["T"], s["lens"], s["path"], s["n_acc"], s["lens_new"])
        return {"path": s["path"], "n_acc": s["n_acc"], "next": s["next"], "lens": s["lens_new"],
                **_state(s)}
    D.kv_evict_q8(s["kv"], s["lens"], c["budget"], c["sink"], c["recent"], s["map"], s["lens_out"],
                  acc_out=s["acc_out"], tpos_out=s["tpos_out"])
    return {"map": s["map"], "lens": s["lens_out"], "acc": s["acc_out"], "tpos": s["tpos_out"],
            **_state(s)}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    """The attention and the accumulated weights from their definition in 64
    bits, one sequence and KV head at a time.  The int8 query is part of the
    definition: q8 = rint(q * (127 / max|q|)) in 32-bit steps.  Moves have
    no computed floating outputs."""
    c = case
    if c["op"] in ("accept", "evict"):
        return None
    s = prepare(c, seed)
    B, T, kvh, hd, H = c["B"], _nodes(c), c["kvh"], c["hd"], c["heads"]
    G, ring, w = H // kvh, _ring(c), c.get("window", 0)
    out = torch.zeros(B * T, H, hd, dtype=torch.float64, device="cuda")
    lse = torch.zeros(B * T, H, dtype=torch.float64, device="cuda")
    acc = s["acc"].double() if "acc" in s else None
    for b, n in enumerate(_lens(c)):
        first = max(0, n + T - ring) if ring else 0
        t = torch.arange(first, n + T, device="cuda")  # positions the cache holds
        slot = t % ring if ring else t
        node = t - n
        vis = (node < 0).expand(T, -1).clone()
        if "see" in s:
            vis[:, node >= 0] = s["see"][b][:, node[node >= 0]]
        else:
            vis[:, node >= 0] = True
        if w:
            pos = s["pos"].reshape(B, T)[b].long()
            at = t.clone()
            at[node >= 0] = pos[node[node >= 0]]
            vis &= at[None] > pos[:, None] - w
        sum_w = torch.zeros(len(t), dtype=torch.float64, device="cuda")
        for k in range(kvh):
            key = s["kc"][b, slot, k * hd:(k + 1) * hd].double() * s["ks"][b, slot].double()[:, None]
            val = s["vt"][b, slot // 4, k * hd:(k + 1) * hd, slot % 4].double()
            val = val * s["vs"][b, slot].double()[:, None]
            for g in range(G):
                h = k * G + g
                q = s["q"][b * T:(b + 1) * T, h * hd:(h + 1) * hd].cpu().numpy()
                top = np.abs(q).max(-1, keepdims=True)
                inv = np.divide(np.float32(127), top, out=np.zeros_like(top), where=top > 0)
                q8 = np.clip(np.rint(q * inv), -127, 127).astype(np.float64)
                q8 = q8 * (top / np.float32(127)).astype(np.float64)
                sc = torch.from_numpy(q8).cuda() @ key.T
                sc[~vis] = -math.inf
                if c["op"] == "accum":
                    p = torch.exp(sc - s["lse"][b * T:(b + 1) * T, h].double()[:, None])
                    sum_w += (p * s["take"][b].double()[:, None]).sum(0)
                    continue
                top_s = sc.amax(-1, keepdim=True)
                p = torch.exp(sc - top_s)
                l = p.sum(-1, keepdim=True)
                out[b * T:(b + 1) * T, h] = (p / l) @ val
                lse[b * T:(b + 1) * T, h] = (top_s + torch.log(l))[:, 0]
                sum_w += (p / l).sum(0)
        if acc is not None:
            acc[b, slot] = torch.where(node < 0, DECAY * acc[b, slot], 0.0) + sum_w
    if c["op"] == "accum":
        return {"acc": acc}
    if c["op"] == "decode":
        return {"out": out.flatten(1), "acc": acc}
    return {"out": out.flatten(1), "lse": lse}
