"""The KV-cache operators where their kernels divide or reorder the work in
ways that short random cases do not reach.  Helpers, caches and tolerances are
those of test_kv_tree.py."""
import numpy as np
import pytest

import fastgemma_b200.device as D
from test_kv_tree import EPS, Cache, accum64, attend64, check_attend, dev, run_attend, setup

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


# ------------------------------------- maxima that grow all along a long run
def staircases(rng, rows, T, H, kvh, hd, tiles):
    """Scores by tile of 128 slots: a query row's rises by 7 levels a tile up
    to a tile of its own and stays there.  K holds 127 in the dimension of the
    slot's tile, q the row's level there (and 127 where K holds 0, which makes
    the int8 query the levels themselves), and a level is 9 ln 2 / 7, so that
    one step multiplies the weights by 2^9."""
    n = tiles * 128 - T
    cache = Cache(rng, rows, n + T, kvh, hd)
    k = cache.k.reshape(rows, n + T, kvh, hd)
    k[..., :tiles] = k[..., -1:] = 0
    for x in range(n + T):
        k[:, x, :, x // 128] = 127
    cache.ks[:] = 9 * np.log(2) / 7 / 127 * rng.uniform(0.99, 1.01, cache.ks.shape)
    level = np.arange(tiles) * 7
    stop = (np.arange(rows * T * H) * 5 % tiles).reshape(rows * T, H)
    q = np.zeros((rows * T, H, hd), np.float32)
    q[..., :tiles] = np.minimum(level, level[stop][..., None])
    q[..., -1] = 127
    pos = np.tile(n + np.arange(T, dtype=np.int32), (rows, 1))
    return cache, q.reshape(rows * T, -1), [n] * rows, pos


@gpu
@pytest.mark.parametrize("rows,T,H,kvh,hd,tiles", [(16, 16, 64, 8, 64, 16),  # a CTA an item
                                                   (16, 64, 8, 4, 256, 16),
                                                   (3, 33, 16, 4, 320, 17),
                                                   (8, 128, 4, 4, 512, 16),
                                                   (37, 20, 4, 4, 128, 16)])
def test_maxima_that_grow_in_every_tile(rows, T, H, kvh, hd, tiles):
    """In every tile some rows of each warp rescale their output and others
    keep all that it holds: the rescaling has to come before the products."""
    rng = np.random.default_rng(hd)
    cache, q, lens, pos = staircases(rng, rows, T, H, kvh, hd, tiles)
    (kv, qd, ld, _, pd, out, lse), _, _ = check_attend(cache, q, H, T, lens, None, pos, 0)
    ws = D.attend_workspace(kv, H, T)
    again, lse2 = torch.empty_like(qd), torch.empty_like(lse)
    for _ in range(50):
        D.attend_tree_q8(again, qd, kv, H, T, ld, pos=pd, lse=lse2, ws=ws)
        assert torch.equal(again, out) and torch.equal(lse2, lse)


# ------------------------------------------------- nodes that add nothing
@gpu
@pytest.mark.parametrize("T,H,kvh,hd,kind", [(2, 4, 2, 64, "chain"), (48, 8, 2, 128, "tree"),
                                             (150, 4, 2, 320, "chain")])
def test_a_node_that_is_not_taken_adds_nothing_whatever_its_query_holds(T, H, kvh, hd, kind):
    """Rejected nodes with a not-a-number and an infinity in a query head: the
    slots' weights have the bits they have with finite queries there."""
    rng = np.random.default_rng(T)
    lens = [300, 77]
    cache, q, mask, pos = setup(rng, lens, T, H, kvh, hd, kind)
    take = rng.integers(0, 2, (2, T)).astype(np.uint8)
    take[:, 1], take[:, 0] = 0, 1
    got = []
    for bad in (False, True):
        if bad:
            q[1, 3] = np.nan
            q[T + 1, hd:] = np.inf
        kv, qd, ld, w, pd, _, lse = run_attend(cache, q, H, T, lens, mask, pos, 0)
        D.attend_accum_q8(qd, kv, H, T, ld, lse, mask=w, pos=pd, take=dev(take), decay=0.5)
        got.append(cache.d["acc"].cpu().numpy())
    assert np.isfinite(got[0]).all()
    assert np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32))


# --------------------------------------- tensors that would be misread
def test_rows_of_another_type_or_stride_are_refused():
    T, H, kvh, hd, cap = 3, 4, 2, 64, 12
    kc, s = torch.zeros(2, cap, kvh * hd, dtype=torch.int8), torch.zeros(2, cap)
    kv = D.KvCache(kc, s, kc.reshape(2, -1), s, kvh, hd, acc=torch.zeros(2, cap))
    lens = torch.zeros(2, dtype=torch.int32)
    q, ws = torch.zeros(2 * T, H * hd), torch.zeros(1, dtype=torch.uint8)
    lse, one = torch.zeros(2 * T, H), torch.zeros(2, H * hd)

    def refused(name, f, *a, **kw):
        with pytest.raises(ValueError, match=name):
            f(*a, ws=ws, **kw)

    for bad in (q.bfloat16(), q.double(), torch.zeros(2 * T, H * hd, 2)[..., 0]):
        refused("^q ", D.attend_tree_q8, q, bad, kv, H, T, lens)
        refused("^out ", D.attend_tree_q8, bad, q, kv, H, T, lens)
        refused("^q ", D.attend_accum_q8, bad, kv, H, T, lens, lse)
        refused("^q ", D.attend_acc_q8, one, bad[:2], kv, H, lens)
        refused("^out ", D.attend_acc_q8, bad[:2], one, kv, H, lens)
    for bad in (lse.double(), lse.half(), lse[:5], lse[:, :3], lse.reshape(2, T, H), lse.flatten()):
        refused("^lse", D.attend_tree_q8, q, q, kv, H, T, lens, lse=bad)
        refused("^lse", D.attend_accum_q8, q, kv, H, T, lens, bad)

    m = torch.zeros(2, 8, dtype=torch.int32)
    acc, tpos = torch.zeros(2, 8), torch.zeros(2, 8, dtype=torch.int32)
    for bad in (acc.double(), tpos, acc[:1], acc[:, :7], acc.flatten(), torch.zeros(8, 2).t(),
                torch.zeros(2, 16)[:, ::2]):
        with pytest.raises(ValueError, match="^acc_out"):
            D.kv_evict_q8(kv, lens, 8, 1, 1, m, lens, acc_out=bad)
    for bad in (tpos.long(), acc, tpos[:1], tpos[:, :7]):
        with pytest.raises(ValueError, match="^tpos_out"):
            D.kv_evict_q8(kv, lens, 8, 1, 1, m, lens, tpos_out=bad)

    k, pos = torch.zeros(2 * T, kvh * hd), torch.zeros(2 * T, dtype=torch.int32)
    w = torch.zeros(hd)
    for name, a in (("q", (q.double(), k, k)), ("k", (q, k.half(), k)), ("v", (q, k, k.bfloat16()))):
        with pytest.raises(ValueError, match=f"^{name} "):
            D.qkv_post_tree(kv, *a, H, T, w, w, 1e-6, w, pos, lens)


# ------------------------------------------------ nodes into the cache
@gpu
@pytest.mark.parametrize("lens,T,H,kvh,hd,ring,q_pad,kv_pad", [
    ([0], 1, 1, 1, 64, 0, 0, 0), ([50, 0, 37], 7, 8, 2, 256, 0, 12, 4), ([61, 10], 33, 4, 4, 128, 0, 0, 8),
    ([100, 3], 20, 8, 1, 512, 33, 4, 0), ([9], 256, 16, 2, 192, 0, 0, 0),
    ([1000, 40], 40, 12, 3, 320, 40, 8, 8)])
def test_chain_rows_need_no_positions(lens, T, H, kvh, hd, ring, q_pad, kv_pad):
    """qkv_post_tree without positions against the same with lens + i, and both
    against qkv_post with a cache per row; rows further apart than they are long."""
    rng = np.random.default_rng(T + hd)
    rows, n = len(lens), len(lens) * T
    cap = ring + 2 if ring else max(lens) + T - 3 if T > 3 else max(lens) + T  # some past the end
    pos = (np.array(lens, np.int32)[:, None] + np.arange(T, dtype=np.int32)).reshape(-1)
    ld = dev(np.array(lens, np.int32))
    qn, kn = (dev(rng.uniform(0.5, 1.5, hd).astype(np.float32)) for _ in range(2))
    inv = (1.0 / 10000.0 ** (np.arange(0, hd, 2) / hd)).astype(np.float32)
    cs = dev(D.rope_table(60, hd, inv))  # shorter than the positions
    x = [rng.standard_normal((n, w)).astype(np.float32)
         for w in (H * hd + q_pad, kvh * hd + kv_pad, kvh * hd + kv_pad)]
    got = []
    for p in (dev(pos), None):
        c = Cache(np.random.default_rng(1), rows, cap, kvh, hd, ring)
        kv = c.put()
        a = [dev(t) for t in x]
        D.qkv_post_tree(kv, *a, H, T, qn, kn, 1e-6, dev(inv), p, ld, q_ld=H * hd + q_pad,
                        kv_ld=kvh * hd + kv_pad, cs=cs)
        got.append((a, c))
    (a, c), (a2, c2) = got
    assert all(torch.equal(s, t) for s, t in zip(a, a2))
    assert all(torch.equal(c.d[k].view(torch.uint8), c2.d[k].view(torch.uint8)) for k in c.d)
    # one cache per row, the slot being the position (0 where it is past 300)
    each = Cache(rng, n, 300, kvh, hd)
    each.put()
    d, at, w = each.d, np.where(pos < 300, pos, 0), [dev(t) for t in x]
    D.qkv_post(*w, n, H, kvh, hd, qn, kn, 1e-6, dev(inv), dev(pos), 0, 300, d["kc"],
               d["kc"].stride(0), d["ks"], 300, d["vt"], d["vt"].stride(0), d["vs"], 300, cs=cs,
               q_ld=H * hd + q_pad, kv_ld=kvh * hd + kv_pad)
    assert all(torch.equal(s, t) for s, t in zip(a, w))
    kd = d["kc"].cpu().numpy()
    vt = d["vt"].cpu().numpy().reshape(n, 75, kvh * hd, 4)
    ks, vs = d["ks"].cpu().numpy(), d["vs"].cpu().numpy()
    sure = np.zeros((rows, cap), bool)  # slots whose row the caches per row can tell
    sure[:] = True
    for r in range(n):
        s = pos[r] % ring if ring else pos[r]
        if s >= cap:
            continue
        sure[r // T, s] = pos[r] < 300
        p = at[r]
        c.k[r // T, s], c.v[r // T, s] = kd[r, p], vt[r, p // 4, :, p % 4]
        c.ks[r // T, s], c.vs[r // T, s], c.tpos[r // T, s] = ks[r, p], vs[r, p], pos[r]
    assert np.array_equal(c.d["kc"].cpu().numpy()[sure], c.k[sure])
    got_v = c.d["vt"].cpu().numpy().reshape(rows, -1, kvh * hd, 4).transpose(0, 1, 3, 2)
    assert np.array_equal(got_v.reshape(rows, -1, kvh * hd)[:, :cap][sure], c.v[:, :cap][sure])
    for name in ("ks", "vs"):
        assert np.array_equal(c.d[name].cpu().numpy()[sure], getattr(c, name)[sure])
    assert np.array_equal(c.d["tpos"].cpu().numpy(), c.tpos)


# --------------------------------------------------------- large batches
def many(rng, rows, most):
    """Lengths of every size up to `most`, among them 0 and `most`."""
    lens = np.exp(rng.uniform(0, np.log(most), rows)).astype(int)
    lens[rows // 2], lens[-1] = 0, most
    return lens.tolist()


@gpu
@pytest.mark.parametrize("rows,T,H,kvh,hd,kind,window,most", [
    (33, 2, 4, 2, 64, "tree", 0, 700), (64, 3, 8, 4, 128, "chain", 0, 2500),
    (100, 1, 2, 1, 256, "chain", 50, 300), (70, 5, 8, 2, 64, "tree", 90, 1500),
    (33, 20, 4, 2, 64, "tree", 0, 1500), (64, 40, 8, 8, 64, "any", 0, 400),
    (70, 33, 2, 1, 128, "tree", 120, 1300), (40, 17, 2, 2, 320, "chain", 0, 600)])
def test_batches_of_more_sequences_than_a_warp_has_lanes(rows, T, H, kvh, hd, kind, window, most):
    """Ragged batches, from fewer items than SMs to several times as many, with
    few and with many query rows per KV head; attention, then its weights."""
    rng = np.random.default_rng(rows * T + hd)
    lens = many(rng, rows, most)
    cache, q, mask, pos = setup(rng, lens, T, H, kvh, hd, kind, window)
    (kv, qd, ld, w, pd, _, lse), weights, S = check_attend(cache, q, H, T, lens, mask, pos, window)
    take = rng.integers(0, 2, (rows, T)).astype(np.uint8)
    want = accum64(cache, weights, T, lens, take, np.float32(0.9), None)
    D.attend_accum_q8(qd, kv, H, T, ld, lse, mask=w, pos=pd, window=window, take=dev(take), decay=0.9)
    got = cache.d["acc"].cpu().numpy()
    tol = (32 * S + 128 + (most + T) / 8 + T * H) * EPS
    assert (np.abs(got - want) <= tol * np.maximum(np.abs(want), 1)).all()
    for b, n in enumerate(lens):
        assert np.array_equal(got[b, n + T:], cache.acc[b, n + T:])


@gpu
@pytest.mark.parametrize("rows,H,kvh,hd,most", [(33, 4, 2, 64, 900), (100, 8, 1, 256, 300),
                                                (70, 16, 4, 128, 1500)])
def test_decode_step_of_more_sequences_than_a_warp_has_lanes(rows, H, kvh, hd, most):
    rng = np.random.default_rng(rows)
    lens = many(rng, rows, most)
    cache, q, _, pos = setup(rng, lens, 1, H, kvh, hd, "chain")
    want, _, weights, S, V = attend64(cache, q, H, 1, lens, None, pos, 0)
    kv, out = cache.put(), torch.empty(rows, H * hd, device="cuda")
    D.attend_acc_q8(out, dev(q), kv, H, dev(np.array(lens, np.int32)), decay=0.75)
    tol = (16 * S + 64 + (most + 1) / 8) * EPS
    assert np.abs(out.cpu().numpy() - want).max() <= tol * V
    acc = accum64(cache, weights, 1, lens, None, 0.75, None)
    got = cache.d["acc"].cpu().numpy()
    assert (np.abs(got - acc) <= (2 * tol + H * EPS) * np.maximum(acc, 1)).all()


@gpu
@pytest.mark.parametrize("T", [1, 17])
def test_more_items_than_a_launch_splits(T):
    """130 sequences of 128 KV heads: an item a CTA, whatever its length."""
    rng = np.random.default_rng(T)
    rows, H, hd, most = 130, 128, 64, 140
    lens = many(rng, rows, most)
    cache, q, _, pos = setup(rng, lens, T, H, H, hd, "chain")
    kv, qd, ld, _, pd, out, lse = run_attend(cache, q, H, T, lens, None, pos, 0)
    want, wlse, acc = np.zeros((rows * T, H, hd)), np.zeros((rows * T, H)), cache.acc.astype(float)
    S = V = 0.0
    for b, n in enumerate(lens):
        qb = q[b * T:(b + 1) * T].reshape(T, H, hd)
        top = np.abs(qb).max(-1, keepdims=True)
        q8 = np.clip(np.rint(qb * (np.float32(127) / top)), -127, 127).astype(np.float64)
        k = cache.k[b, :n + T].reshape(-1, H, hd) * cache.ks[b, :n + T, None, None].astype(float)
        v = cache.v[b, :n + T].reshape(-1, H, hd) * cache.vs[b, :n + T, None, None].astype(float)
        s = np.einsum("thd,nhd->thn", q8 * (top / np.float32(127)).astype(float), k)
        s[~np.broadcast_to((np.arange(n + T) <= n + np.arange(T)[:, None])[:, None], s.shape)] = -np.inf
        m = s.max(-1, keepdims=True)
        e = np.exp(s - m)
        p = e / e.sum(-1, keepdims=True)
        want[b * T:(b + 1) * T] = np.einsum("thn,nhd->thd", p, v)
        wlse[b * T:(b + 1) * T] = (m + np.log(e.sum(-1, keepdims=True)))[..., 0]
        acc[b, :n + T] = np.where(np.arange(n + T) < n, 0.5 * acc[b, :n + T], 0) + p.sum((0, 1))
        S, V = max(S, np.abs(s[np.isfinite(s)]).max()), max(V, np.abs(v).max())
    tol = (16 * S + 64 + (most + T) / 8) * EPS
    assert np.abs(out.cpu().numpy() - want.reshape(rows * T, -1)).max() <= tol * V
    assert (np.abs(lse.cpu().numpy() - wlse) <= tol * np.maximum(1, np.abs(wlse))).all()
    bound = (2 * tol + T * H * EPS) * np.maximum(acc, 1)
    D.attend_accum_q8(qd, kv, H, T, ld, lse, pos=pd, decay=0.5)
    assert (np.abs(cache.d["acc"].cpu().numpy() - acc) <= bound).all()
    if T == 1:
        cache.d["acc"].copy_(dev(cache.acc))
        one = torch.empty_like(qd)
        D.attend_acc_q8(one, qd, kv, H, ld, decay=0.5)
        assert np.abs(one.cpu().numpy() - want.reshape(rows, -1)).max() <= tol * V
        assert (np.abs(cache.d["acc"].cpu().numpy() - acc) <= bound).all()


# ----------------------------------------------------- sums over long runs
@gpu
@pytest.mark.parametrize("T,tol", [(1, 2 * 34 + 16), (3, 2 * 17 * 33 + 16)])
def test_long_sums_are_not_rounded_towards_zero(T, tol):
    """Equal weights over positive values, every item of 128 on one CTA: sums
    that grow all along.  An instruction of the tensor cores may cut each of its
    16 products and what it adds them to down to 2^-23 of the sum, 17 units, so an
    accumulator that takes all of a run loses a part that grows with the run.
    Rounding to nearest has no mean error; what the mean over all outputs may be
    off is the units of two instructions on one step's sum (streaming kernel), or
    of 64 on the growing sum of four tiles (tile kernel, 17 * 33 units), and 16 *
    2^-24 for the weights' 22 bits, the division and the scaling.  The sum of
    the weights is exact."""
    n = 65536
    g = torch.Generator(device="cuda").manual_seed(n)
    rows, kvh, G, hd, cap = 16, 8, 8, 64, n + 4
    kvd = kvh * hd
    kc = torch.zeros(rows, cap, kvd, dtype=torch.int8, device="cuda")
    vt = torch.randint(64, 128, (rows, cap // 4, kvd, 4), dtype=torch.int8, device="cuda", generator=g)
    ks = torch.ones(rows, cap, device="cuda")
    vs = torch.rand(rows, cap, device="cuda", generator=g) * 0.5 + 0.5
    kv = D.KvCache(kc, ks, vt, vs, kvh, hd, acc=torch.zeros(rows, cap, device="cuda"))
    q = torch.zeros(rows * T, kvh * G * hd, device="cuda")
    lens = torch.full((rows,), n, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    D.attend_tree_q8(out, q, kv, kvh * G, T, lens)
    got = out.double().reshape(rows, T, kvh, G, hd)
    want = torch.empty(rows, T, kvd, dtype=torch.float64, device="cuda")
    for b in range(rows):
        x = vt[b].double() * vs[b].double().reshape(-1, 1, 4)
        x = x.transpose(1, 2).reshape(cap, kvd)
        for i in range(T):
            want[b, i] = x[:n + i + 1].sum(0) / (n + i + 1)
    off = got / want.reshape(rows, T, kvh, 1, hd) - 1
    assert abs(off.mean().item()) <= tol * EPS
    if T == 1:
        one = torch.empty_like(q)
        D.attend_acc_q8(one, q, kv, kvh * G, lens)
        off = one.double().reshape(got.shape) / want.reshape(rows, T, kvh, 1, hd) - 1
        assert abs(off.mean().item()) <= tol * EPS
