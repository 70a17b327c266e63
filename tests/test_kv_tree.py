"""Attention of several tokens per sequence over the int8 KV cache, the
weights it accumulates per slot, and the moves of cache rows (verification,
commit, eviction), against plain implementations in 64 bits.

Tolerances.  q . k is a whole number, so a score carries the roundings of its
two scales and two products, 4 * S * 2^-24 for scores up to S, and its
exponential the rounding of its argument and of the exponential itself: a
weight's relative error is at most (8 S + 16) * 2^-24.  An output is a ratio
of sums of such weights, each of up to n terms added in 32 bits in chains of
n / 8 at most: (16 S + 64 + n / 8) * 2^-24 times the largest |vs * v|.  lse
has the weights' error in its logarithm's argument, an accumulated weight the
weights' error times their sum and a rounding per added term."""
import ctypes as C

import numpy as np
import pytest

import fastgemma_b200.device as D
from fastgemma_b200 import _lib

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
EPS = 2.0 ** -24


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ------------------------------------------------------------- plain forms
class Cache:
    """Host copy of one layer's caches; slots nothing was written to hold
    not-a-number scales and arbitrary bytes."""

    def __init__(self, rng, rows, cap, kvh, hd, ring=0):
        self.rows, self.cap, self.kvh, self.hd, self.ring = rows, cap, kvh, hd, ring
        kvd = kvh * hd
        self.k = rng.integers(-127, 128, (rows, cap, kvd)).astype(np.int8)
        self.v = rng.integers(-127, 128, (rows, (cap + 3) // 4 * 4, kvd)).astype(np.int8)
        self.ks = rng.uniform(0.001, 0.02, (rows, cap)).astype(np.float32)
        self.vs = rng.uniform(0.001, 0.02, (rows, cap)).astype(np.float32)
        self.acc = rng.uniform(0, 4, (rows, cap)).astype(np.float32)
        self.tpos = np.tile(np.arange(cap, dtype=np.int32), (rows, 1))

    def forget_past(self, ends):
        for b, e in enumerate(ends):
            if not self.ring:
                self.ks[b, e:] = self.vs[b, e:] = np.nan
            else:
                self.ks[b, min(e, self.ring):] = self.vs[b, min(e, self.ring):] = np.nan

    def vt(self):
        r, n, kvd = self.v.shape
        return np.ascontiguousarray(self.v.reshape(r, n // 4, 4, kvd).transpose(0, 1, 3, 2))

    def put(self, pad=0):
        """Device tensors and their view; pad: slots between one sequence's rows and the next."""
        def spread(a):
            a = a.reshape(a.shape[0], -1)
            per = a.shape[1] // self.cap if a.shape[1] % self.cap == 0 else 1
            t = torch.zeros(a.shape[0], a.shape[1] + pad * max(per, 1) * 16, dtype=dev(a).dtype,
                            device="cuda")
            t[:, :a.shape[1]] = dev(a)
            return t[:, :a.shape[1]]
        self.d = dict(kc=spread(self.k).unflatten(1, (self.cap, -1)), ks=spread(self.ks),
                      vt=spread(self.vt()), vs=spread(self.vs), acc=spread(self.acc),
                      tpos=spread(self.tpos))
        return D.KvCache(self.d["kc"], self.d["ks"], self.d["vt"], self.d["vs"], self.kvh, self.hd,
                         ring=self.ring, acc=self.d["acc"], tpos=self.d["tpos"])

    def same_as_device(self):
        assert np.array_equal(self.d["kc"].cpu().numpy(), self.k)
        vt = self.d["vt"].cpu().numpy().reshape(self.vt().shape)
        assert np.array_equal(vt, self.vt())
        for name in ("ks", "vs", "acc", "tpos"):
            a, b = self.d[name].cpu().numpy(), getattr(self, name)
            assert np.array_equal(a.view(np.uint32), b.view(np.uint32)), name


def positions(cache, n, T):
    """(position, slot) pairs that hold something after n committed tokens and T nodes."""
    first = max(0, n + T - cache.ring) if cache.ring else 0
    t = np.arange(first, n + T)
    return t, (t % cache.ring if cache.ring else t)


def visible(mask, pos, b, n, T, t, window):
    """Bool [T][len(t)]."""
    vis = np.zeros((T, len(t)), bool)
    at = np.array([pos[b, x - n] if x >= n else x for x in t], np.int64)
    for i in range(T):
        among = mask[b, i] if mask is not None else np.arange(T) <= i
        vis[i] = [(x < n) or among[x - n] for x in t]
        if window:
            vis[i] &= at > int(pos[b, i]) - window
    return vis


def attend64(cache, q, H, T, lens, mask, pos, window):
    """(out, lse, weights [b] -> [T][H][positions], largest score, largest |v|)."""
    hd, G = cache.hd, H // cache.kvh
    out = np.zeros((len(lens) * T, H, hd))
    lse = np.full((len(lens) * T, H), -np.inf)
    smax, vmax, weights = 0.0, 0.0, []
    for b, n in enumerate(lens):
        t, slot = positions(cache, n, T)
        vis = visible(mask, pos, b, n, T, t, window)
        seen = vis.any(0)
        wb = np.zeros((T, H, len(t)))
        for h in range(H):
            d = slice(h // G * hd, (h // G + 1) * hd)
            qh = q[b * T:(b + 1) * T, h * hd:(h + 1) * hd]
            top = np.abs(qh).max(-1, keepdims=True)
            inv = np.divide(np.float32(127), top, out=np.zeros_like(top), where=top > 0)
            q8 = np.clip(np.rint(qh * inv), -127, 127).astype(np.float64)
            qs = (top / np.float32(127)).astype(np.float64)
            ks = np.where(seen, cache.ks[b, slot], 0).astype(np.float64)
            vs = np.where(seen, cache.vs[b, slot], 0).astype(np.float64)
            s = (q8 @ cache.k[b, slot][:, d].astype(np.float64).T) * qs * ks
            v = cache.v[b, slot][:, d].astype(np.float64) * vs[:, None]
            for i in range(T):
                if not vis[i].any():
                    continue
                si = s[i, vis[i]]
                e = np.exp(si - si.max())
                wb[i, h, vis[i]] = e / e.sum()
                out[b * T + i, h] = wb[i, h, vis[i]] @ v[vis[i]]
                lse[b * T + i, h] = si.max() + np.log(e.sum())
                smax = max(smax, np.abs(si).max())
                vmax = max(vmax, np.abs(v[vis[i]]).max())
        weights.append(wb)
    return out.reshape(len(lens) * T, -1), lse, weights, smax, vmax


def accum64(cache, weights, T, lens, take, decay, b_lse):
    acc = cache.acc.astype(np.float64)
    for b, n in enumerate(lens):
        t, slot = positions(cache, n, T)
        add = sum(weights[b][i].sum(0) for i in range(T) if take is None or take[b, i]) \
            if take is None or take[b].any() else 0.0
        acc[b, slot] = np.where(t < n, decay * acc[b, slot], 0.0) + add
    return acc


def words(mask):
    bits = np.packbits(mask, axis=-1, bitorder="little")
    bits = np.pad(bits, ((0, 0), (0, 0), (0, -bits.shape[-1] % 8)))
    return np.ascontiguousarray(bits).view(np.int64)


def random_tree(rng, rows, T, reach=4):
    parent = np.full((rows, T), -1, np.int32)
    see = np.zeros((rows, T, T), bool)
    depth = np.zeros((rows, T), np.int32)
    for b in range(rows):
        for i in range(T):
            if i:
                parent[b, i] = rng.integers(max(0, i - reach), i)
                see[b, i] = see[b, parent[b, i]]
                depth[b, i] = depth[b, parent[b, i]] + 1
            see[b, i, i] = True
    return parent, see, depth


def setup(rng, lens, T, H, kvh, hd, kind="tree", window=0, ring=0, extra=5, scale=1.0):
    rows = len(lens)
    cap = ring or max(lens) + T + extra
    cache = Cache(rng, rows, cap, kvh, hd, ring)
    cache.forget_past([n + T for n in lens])
    q = (rng.standard_normal((rows * T, H * hd)) * scale).astype(np.float32)
    depth = np.tile(np.arange(T, dtype=np.int32), (rows, 1))
    mask = None
    if kind == "tree":
        _, mask, depth = random_tree(rng, rows, T)
    elif kind == "any":
        mask = rng.integers(0, 2, (rows, T, T)).astype(bool)
        mask[:, ::3] = False  # every third node sees no node at all
    pos = np.asarray(lens, np.int32)[:, None] + depth
    return cache, q, mask, pos


def run_attend(cache, q, H, T, lens, mask, pos, window, pad=0, q_pad=0, **kw):
    kv = cache.put(pad)
    width = H * cache.hd
    qd = torch.full((q.shape[0], width + q_pad), float("nan"), device="cuda")
    qd[:, :width] = dev(q)
    out = torch.full((q.shape[0], width + q_pad), 7.0, device="cuda")
    lse = torch.full((q.shape[0], H), 7.0, device="cuda")
    w = None if mask is None else dev(words(mask))
    ld = dev(np.asarray(lens, np.int32))
    pd = None if pos is None else dev(pos)
    D.attend_tree_q8(out, qd, kv, H, T, ld, mask=w, pos=pd, window=window, lse=lse,
                     q_ld=width + q_pad, out_ld=width + q_pad, **kw)
    torch.cuda.synchronize()
    assert (out[:, width:] == 7.0).all()
    return kv, qd, ld, w, pd, out[:, :width], lse


def check_attend(cache, q, H, T, lens, mask, pos, window, **kw):
    got = run_attend(cache, q, H, T, lens, mask, pos, window, **kw)
    want, wlse, weights, S, V = attend64(cache, q, H, T, lens, mask, pos, window)
    n = max(lens) + T
    out, lse = got[5].cpu().numpy(), got[6].cpu().numpy()
    tol = (16 * S + 64 + n / 8) * EPS
    assert np.abs(out - want).max() <= tol * V
    empty = np.isneginf(wlse)
    assert np.array_equal(empty, np.isneginf(lse))
    assert (out.reshape(len(q), H, -1)[empty] == 0).all()
    lse, wlse = lse[~empty], wlse[~empty]
    assert (np.abs(lse - wlse) <= tol * np.maximum(1, np.abs(wlse))).all()
    return got, weights, S


# -------------------------------------------------------------- attention
SHAPES = [
    # lens, T, heads, kv heads, head_dim, mask, window, ring
    ([0], 1, 1, 1, 64, "chain", 0, 0),
    ([0, 3], 2, 2, 1, 64, "chain", 0, 0),
    ([1], 1, 8, 2, 256, "chain", 0, 0),
    ([100, 0, 37], 4, 8, 2, 256, "tree", 0, 0),
    ([15, 16, 17], 5, 8, 1, 128, "tree", 0, 0),
    ([127, 128, 129], 1, 4, 4, 192, "chain", 0, 0),
    ([700, 5], 3, 16, 1, 320, "tree", 0, 0),
    ([333], 8, 2, 2, 384, "any", 0, 0),
    ([260, 130], 7, 8, 8, 448, "any", 0, 0),
    ([1023], 16, 8, 2, 512, "tree", 0, 0),
    ([0, 200], 33, 8, 2, 128, "any", 0, 0),
    ([511, 64], 64, 8, 2, 256, "tree", 0, 0),
    ([90], 65, 4, 1, 64, "any", 0, 0),
    ([300], 129, 16, 1, 64, "tree", 0, 0),
    ([77, 0], 256, 4, 2, 256, "chain", 0, 0),
    ([129], 256, 2, 1, 512, "tree", 0, 0),
    ([1500], 130, 4, 1, 192, "tree", 0, 0),
    # sliding windows, in linear caches and in rings (wrapped and not)
    ([400, 10, 90], 4, 8, 2, 256, "tree", 64, 0),
    ([400, 10], 40, 4, 2, 128, "any", 20, 0),
    ([1000, 37, 131], 9, 8, 2, 256, "tree", 64, 72),
    ([500, 3], 60, 8, 2, 128, "tree", 100, 160),
    ([640, 0], 100, 2, 1, 320, "chain", 29, 131),
    ([10000], 1, 8, 2, 256, "chain", 33, 33),
    ([2000, 37, 290], 20, 8, 2, 256, "tree", 280, 300),
    ([3000], 30, 4, 2, 64, "any", 1000, 1100),
    ([700, 5], 70, 2, 1, 512, "chain", 230, 300),
]
# slots past the nodes: many rows over a cache with room take another kernel
# than over one that is short
ROOM = [5, 1200]


@gpu
@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("lens,T,H,kvh,hd,kind,window,ring", SHAPES)
def test_attend_tree(lens, T, H, kvh, hd, kind, window, ring, room):
    rng = np.random.default_rng(sum(lens) * 7 + T * 31 + H + hd)
    cache, q, mask, pos = setup(rng, lens, T, H, kvh, hd, kind, window, ring, room)
    check_attend(cache, q, H, T, lens, mask, pos, window)


@gpu
@pytest.mark.parametrize("T,H,kvh,hd,room", [(3, 8, 2, 256, 5), (40, 8, 2, 64, 5),
                                             (40, 8, 2, 64, 1200), (70, 4, 1, 320, 200)])
def test_attend_strides_and_flat_or_peaked_scores(T, H, kvh, hd, room):
    """Rows and sequences further apart than they are long; a zero query (all
    weights equal) and one slot that takes all the weight."""
    rng = np.random.default_rng(T)
    lens = [150, 149]
    cache, q, mask, pos = setup(rng, lens, T, H, kvh, hd, extra=room)
    q[1] = 0.0
    q[2] *= 40.0
    check_attend(cache, q, H, T, lens, mask, pos, 0, pad=3, q_pad=12)


@gpu
@pytest.mark.parametrize("T,room", [(2, 5), (20, 5), (20, 1200)])
def test_attend_scales_of_every_size(T, room):
    """V scales from 1e-30 to 1e30 and zero, negative K and V scales: the
    weights keep their precision whatever the scales' range."""
    rng = np.random.default_rng(2)
    lens, H, kvh, hd = [300], 8, 2, 128
    for lo, hi in ((-30, -28), (28, 30), (-3, 3)):
        cache, q, mask, pos = setup(rng, lens, T, H, kvh, hd, scale=0.2, extra=room)
        n = 300 + T
        cache.vs[:, :n] = (10.0 ** rng.uniform(lo, hi, n) * rng.choice([1, -1, 0], n))
        cache.ks[:, ::2] *= -1
        check_attend(cache, q, H, T, lens, mask, pos, 0)


@gpu
@pytest.mark.parametrize("T,H,kvh,hd,room", [(3, 8, 2, 256, 5), (20, 8, 2, 128, 1200),
                                             (60, 8, 2, 256, 600)])
def test_one_v_scale_far_above_the_others(T, H, kvh, hd, room):
    """A slot of zeros whose scale is 2^13 times the smallest other: the others
    keep 17 bits of their weights, so half a unit of the 17th is the error that
    joins an output's."""
    rng = np.random.default_rng(T)
    lens = [300, 77]
    cache, q, mask, pos = setup(rng, lens, T, H, kvh, hd, extra=room)
    cache.vs[:, 7] = 0.001 * 2.0 ** 13
    cache.v[:, 7] = 0
    got = run_attend(cache, q, H, T, lens, mask, pos, 0)
    want, _, _, S, V = attend64(cache, q, H, T, lens, mask, pos, 0)
    tol = (16 * S + 64 + (max(lens) + T) / 8) * EPS + 2.0 ** -18
    assert np.abs(got[5].cpu().numpy() - want).max() <= tol * V


@gpu
@pytest.mark.parametrize("T,hd,room", [(2, 128, 5), (48, 256, 5), (48, 256, 300), (48, 64, 1200)])
def test_a_query_that_is_no_number_stays_in_its_head(T, hd, room):
    rng = np.random.default_rng(5)
    H, kvh, lens = 4, 2, [70]
    cache, q, mask, pos = setup(rng, lens, T, H, kvh, hd, extra=room)
    want = run_attend(cache, q, H, T, lens, mask, pos, 0)
    q[1, hd + 3] = np.nan
    q[0, 2 * hd] = np.inf
    got = run_attend(cache, q, H, T, lens, mask, pos, 0)
    bad = np.zeros((T, H), bool)
    bad[1, 1] = bad[0, 2] = True
    for a, b in ((got[5].reshape(T, H, hd), want[5].reshape(T, H, hd)), (got[6], want[6])):
        a, b = a.cpu().numpy(), b.cpu().numpy()
        assert np.isnan(a[bad]).all()
        assert np.array_equal(a[~bad], b[~bad])


@gpu
@pytest.mark.parametrize("T,cap", [(1, 90), (40, 90), (40, 1100)])
def test_lengths_outside_the_cache_count_as_the_nearest_inside(T, cap):
    rng = np.random.default_rng(6)
    H, kvh, hd = 4, 2, 64
    cache = Cache(rng, 3, cap, kvh, hd)
    q = rng.standard_normal((3 * T, H * hd)).astype(np.float32)
    a = run_attend(cache, q, H, T, [-5, cap - T + 1, 2 ** 31 - 1], None, None, 0)
    b = run_attend(cache, q, H, T, [0, cap - T, cap - T], None, None, 0)
    assert torch.equal(a[5], b[5]) and torch.equal(a[6], b[6])


@gpu
def test_mask_bits_past_the_last_node_do_not_matter():
    rng = np.random.default_rng(7)
    lens, T, H, kvh, hd = [30], 5, 8, 2, 64
    cache, q, mask, pos = setup(rng, lens, T, H, kvh, hd)
    a = run_attend(cache, q, H, T, lens, mask, pos, 0)
    kv, qd, ld, w, pd = a[:5]
    w |= ~((1 << T) - 1)
    out, lse = torch.empty_like(qd), torch.empty(T, H, device="cuda")
    D.attend_tree_q8(out, qd, kv, H, T, ld, mask=w, pos=pd, lse=lse)
    assert torch.equal(out, a[5]) and torch.equal(lse, a[6])


@gpu
def test_attend_past_two_to_the_31_bytes():
    """A cache whose byte offsets pass 32 bits: a window of the last positions
    of 4.2 million."""
    n, T, H, hd, window = 4_200_000, 3, 2, 512, 50
    rng = np.random.default_rng(8)
    cap = n + T + 1
    small = Cache(rng, 1, 64, 1, hd)
    kc = torch.zeros(1, cap, hd, dtype=torch.int8, device="cuda")
    vt = torch.zeros(1, (cap + 3) // 4, hd, 4, dtype=torch.int8, device="cuda")
    ks, vs = (torch.full((1, cap), float("nan"), device="cuda") for _ in range(2))
    slots = torch.arange(n + T - 64, n + T, device="cuda")
    kc[0, slots] = dev(small.k[0])
    vt[0, slots // 4, :, slots % 4] = dev(small.v[0])
    ks[0, slots], vs[0, slots] = dev(small.ks[0]), dev(small.vs[0])
    acc = torch.ones(1, cap, device="cuda")
    kv = D.KvCache(kc, ks, vt, vs, 1, hd, acc=acc)
    q = rng.standard_normal((T, H * hd)).astype(np.float32) * 0.3
    out, lse = torch.empty(T, H * hd, device="cuda"), torch.empty(T, H, device="cuda")
    lens = dev(np.array([n], np.int32))
    D.attend_tree_q8(out, dev(q), kv, H, T, lens, window=window, lse=lse)
    # the same rows at the end of a short cache
    pos = np.arange(64 - T, 64, dtype=np.int32)[None]
    want, wlse, weights, S, V = attend64(small, q, H, T, [64 - T], None, pos, window)
    tol = (16 * S + 64 + 64) * EPS
    assert np.abs(out.cpu().numpy() - want).max() <= tol * V
    D.attend_accum_q8(dev(q), kv, H, T, lens, lse, window=window)
    got = acc[0, slots].cpu().numpy()
    add = weights[0].sum((0, 1))
    exp = np.where(np.arange(64) < 64 - T, 1.0, 0.0) + add
    assert np.abs(got - exp).max() <= tol * T * H
    assert (acc[0, :n - 64] == 1).all() and acc[0, -1] == 1


@gpu
def test_a_chain_agrees_with_the_single_token_attention():
    """attend_q8 on each prefix, up to its 16-bit weights."""
    rng = np.random.default_rng(9)
    n, T, H, kvh, hd = 45, 3, 8, 2, 256
    cache, q, _, pos = setup(rng, [n], T, H, kvh, hd, "chain")
    kv, qd, ld, _, _, out, _ = run_attend(cache, q, H, T, [n], None, pos, 0)
    want, _, weights, S, V = attend64(cache, q, H, T, [n], None, pos, 0)
    for i in range(T):
        one = torch.empty(1, H * hd, device="cuda")
        D.attend_q8(one, H * hd, qd[i], H * hd, cache.d["kc"], 0, cache.d["ks"], 0, cache.d["vt"],
                    0, cache.d["vs"], 0, 1, H, kvh, hd, 0, n + i + 1)
        bound = (n + i + 1) * V * 0.6 / 65535 + (16 * S + 64) * EPS * V
        assert (one[0] - out[i]).abs().max() <= bound


# ------------------------------------------------------ accumulated weights
@gpu
@pytest.mark.parametrize("lens,T,H,kvh,hd,kind,window,ring", SHAPES)
@pytest.mark.parametrize("some", [False, True])
def test_accumulated_weights(lens, T, H, kvh, hd, kind, window, ring, some):
    rng = np.random.default_rng(sum(lens) * 3 + T * 5 + H + hd + some)
    cache, q, mask, pos = setup(rng, lens, T, H, kvh, hd, kind, window, ring, ROOM[some])
    (kv, qd, ld, w, pd, _, lse), weights, S = check_attend(cache, q, H, T, lens, mask, pos, window)
    take = rng.integers(0, 2, (len(lens), T)).astype(np.uint8) if some else None
    want = accum64(cache, weights, T, lens, take, np.float32(0.9), None)
    D.attend_accum_q8(qd, kv, H, T, ld, lse, mask=w, pos=pd, window=window,
                      take=None if take is None else dev(take), decay=0.9)
    got = cache.d["acc"].cpu().numpy()
    n = max(lens) + T
    tol = (32 * S + 128 + n / 8 + T * H) * EPS
    assert (np.abs(got - want) <= tol * np.maximum(np.abs(want), 1)).all()
    for b, m in enumerate(lens):  # slots nothing lies in keep what they held
        if not ring:
            assert np.array_equal(got[b, m + T:], cache.acc[b, m + T:])


@gpu
@pytest.mark.parametrize("lens,H,kvh,hd", [([0], 1, 1, 64), ([1, 0, 15], 8, 2, 256),
                                           ([1000, 999], 8, 2, 256), ([513], 16, 1, 512),
                                           ([300, 5, 77], 12, 4, 192), ([5000], 16, 2, 128),
                                           ([260], 8, 8, 320)])
def test_decode_step_with_accumulation(lens, H, kvh, hd):
    rng = np.random.default_rng(sum(lens) + H + hd)
    cache, q, _, pos = setup(rng, lens, 1, H, kvh, hd, "chain", extra=9)
    want, _, weights, S, V = attend64(cache, q, H, 1, lens, None, pos, 0)
    kv, ld = cache.put(), dev(np.asarray(lens, np.int32))
    out = torch.empty(len(lens), H * hd, device="cuda")
    D.attend_acc_q8(out, dev(q), kv, H, ld, decay=0.75)
    n = max(lens) + 1
    tol = (16 * S + 64 + n / 8) * EPS
    assert np.abs(out.cpu().numpy() - want).max() <= tol * V
    acc = accum64(cache, weights, 1, lens, None, 0.75, None)
    got = cache.d["acc"].cpu().numpy()
    assert (np.abs(got - acc) <= (2 * tol + H * EPS) * np.maximum(acc, 1)).all()
    for b, m in enumerate(lens):
        assert np.array_equal(got[b, m + 1:], cache.acc[b, m + 1:])


@gpu
@pytest.mark.parametrize("T,room", [(3, 5), (50, 5), (50, 1200)])
def test_lse_by_head(T, room):
    """lse as [heads][nodes]: the same values, written and read through its strides."""
    rng = np.random.default_rng(T)
    lens, H, kvh, hd = [140], 8, 2, 64
    cache, q, mask, pos = setup(rng, lens, T, H, kvh, hd, extra=room)
    kv, qd, ld, w, pd, out, lse = run_attend(cache, q, H, T, lens, mask, pos, 0)
    by_head = torch.zeros(H, T, device="cuda").t()
    D.attend_tree_q8(out.clone(), qd, kv, H, T, ld, mask=w, pos=pd, lse=by_head)
    assert torch.equal(by_head, lse)
    D.attend_accum_q8(qd, kv, H, T, ld, lse, mask=w, pos=pd)
    acc = cache.d["acc"].clone()
    cache.d["acc"].copy_(dev(cache.acc))
    D.attend_accum_q8(qd, kv, H, T, ld, by_head, mask=w, pos=pd)
    assert torch.equal(cache.d["acc"], acc)


@gpu
@pytest.mark.parametrize("T", [2, 70])
def test_equal_inputs_give_equal_bits(T):
    rng = np.random.default_rng(11)
    lens, H, kvh, hd = [900, 310, 55], 8, 2, 256
    cache, q, mask, pos = setup(rng, lens, T, H, kvh, hd)
    got = []
    for _ in range(3):
        kv, qd, ld, w, pd, out, lse = run_attend(cache, q, H, T, lens, mask, pos, 0)
        D.attend_accum_q8(qd, kv, H, T, ld, lse, mask=w, pos=pd, decay=0.5)
        acc = cache.d["acc"].clone()
        D.attend_acc_q8(out.clone(), qd, kv, H, ld, decay=0.5)
        got.append((out.clone(), lse, acc, cache.d["acc"].clone()))
    for g in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(g, got[0]))


# ------------------------------------------------------- trees and moves
def walk(parent, token, target):
    path, cur = [0], 0
    while True:
        kids = [i for i in range(cur + 1, len(parent))
                if parent[i] == cur and token[i] == target[cur]]
        if not kids:
            return path, target[cur]
        cur = kids[0]
        path.append(cur)


@gpu
@pytest.mark.parametrize("rows,T", [(1, 1), (3, 2), (2, 31), (4, 32), (3, 33), (2, 64), (5, 100),
                                    (2, 256)])
def test_tree_mask_and_verify(rows, T):
    rng = np.random.default_rng(rows * 1000 + T)
    parent, see, depth = random_tree(rng, rows, T)
    token = rng.integers(0, 3, (rows, T)).astype(np.int32)
    target = rng.integers(0, 3, (rows, T)).astype(np.int32)
    if T > 4:  # nodes that hang nowhere
        parent[0, 3] = 3
        parent[-1, 4] = -7
        for b in (0, rows - 1):  # the masks of the changed trees
            for i in range(T):
                see[b, i], depth[b, i] = False, 0
                p = parent[b, i]
                if 0 <= p < i:
                    see[b, i], depth[b, i] = see[b, p], depth[b, p] + 1
                see[b, i, i] = True
    lens = np.arange(10, 10 + rows, dtype=np.int32)
    mask = torch.full((rows, T, (T + 63) // 64), -1, dtype=torch.int64, device="cuda")
    pos = torch.zeros(rows * T, dtype=torch.int32, device="cuda")
    D.tree_mask(mask, pos, dev(parent), dev(lens))
    assert np.array_equal(mask.cpu().numpy(), words(see))
    assert np.array_equal(pos.cpu().numpy().reshape(rows, T), lens[:, None] + depth)
    path = torch.full((rows, T), 99, dtype=torch.int32, device="cuda")
    n_acc, nxt = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2))
    D.tree_verify(path, n_acc, nxt, dev(parent), dev(token), dev(target))
    for b in range(rows):
        want, after = walk(parent[b], token[b], target[b])
        assert path[b].tolist() == want + [-1] * (T - len(want))
        assert n_acc[b].item() == len(want) and nxt[b].item() == after


@gpu
@pytest.mark.parametrize("rows,T,layers,hd", [(1, 1, 1, 64), (3, 9, 2, 256), (2, 64, 3, 192),
                                              (2, 256, 1, 64), (1, 20, 35, 64)])
def test_accepted_path_moves_behind_the_committed_rows(rows, T, layers, hd):
    """Linear and ring caches of different sizes in one call."""
    rng = np.random.default_rng(T + layers)
    lens = np.array([700 - 31 * b for b in range(rows)], np.int32)
    path = np.full((rows, T), -1, np.int32)
    n_acc = np.zeros(rows, np.int32)
    for b in range(rows):
        take = np.sort(rng.choice(np.arange(1, T), rng.integers(0, T), replace=False)) \
            if T > 1 else np.array([], int)
        path[b, 0] = 0
        path[b, 1:1 + len(take)] = take
        n_acc[b] = 1 + len(take)
    caches, views = [], []
    for layer in range(layers):
        ring = (300 + layer) if layer % 2 else 0
        c = Cache(rng, rows, ring + 3 if ring else 700 + T + layer, 1 + layer % 3, hd, ring)
        caches.append(c)
        views.append(c.put())
    new = torch.zeros(rows, dtype=torch.int32, device="cuda")
    D.kv_accept(D.kv_layers(views), T, dev(lens), dev(path), dev(n_acc), new)
    assert np.array_equal(new.cpu().numpy(), lens + n_acc)
    for c in caches:
        for b in range(rows):
            for j in range(n_acc[b]):
                s, d = lens[b] + path[b, j], lens[b] + j
                s, d = (s % c.ring, d % c.ring) if c.ring else (s, d)
                for a in (c.k, c.v, c.ks, c.vs, c.acc, c.tpos):
                    a[b, d] = a[b, s]
        c.same_as_device()


def evict_plan(acc, tpos, n, budget, sink, recent):
    """The map of one sequence, by sorting."""
    if n <= budget:
        return [x if x < n else -1 for x in range(budget)]
    newest = tpos[:n].max()
    key = []
    for x in range(n):
        safe = tpos[x] < sink or int(tpos[x]) > int(newest) - recent
        bad = np.isnan(acc[x])
        key.append((0 if safe else 1, 1 if bad and not safe else 0,
                    0.0 if safe or bad else -float(acc[x]), x))
    keep = sorted(k[-1] for k in sorted(key)[:budget])
    late = iter([x for x in keep if x >= budget])
    low = set(x for x in keep if x < budget)
    return [x if x in low else next(late) for x in range(budget)]


@gpu
@pytest.mark.parametrize("lens,budget,sink,recent,kind", [
    ([1], 1, 0, 0, "random"), ([5, 0, 2], 3, 1, 1, "random"),
    ([600, 512, 511, 33], 512, 4, 64, "random"), ([1000], 31, 0, 0, "random"),
    ([1000, 1000], 32, 8, 40, "random"), ([777], 500, 4, 600, "random"),
    ([2049, 1500], 1024, 4, 100, "ties"), ([3000], 2999, 0, 7, "equal"),
    ([1025], 1, 0, 0, "nan"), ([4000, 3999], 2000, 4, 32, "nan"),
    ([900], 450, 5, 50, "moved"), ([20000], 15000, 4, 1000, "ties"),
    ([9000, 8193, 40], 8192, 0, 1, "moved"), ([5000, 4999], 2500, 0, 0, "equal"),
    ([400000], 200000, 4, 1000, "ties")])
@pytest.mark.parametrize("in_place", [False, True])
def test_eviction_to_a_budget(lens, budget, sink, recent, kind, in_place):
    rng = np.random.default_rng(sum(lens) + budget + recent)
    rows, cap = len(lens), max(max(lens), budget) + 3
    c = Cache(rng, rows, cap, 2, 64)
    if kind == "ties":
        c.acc = rng.integers(0, 4, c.acc.shape).astype(np.float32)
    elif kind == "equal":
        c.acc[:] = 0.0
        c.acc[:, ::2] = -0.0  # the same weight
    elif kind == "nan":
        c.acc[rng.random(c.acc.shape) < 0.6] = np.nan
        c.acc[:, 7], c.acc[:, 9] = np.inf, -np.inf
    elif kind == "moved":  # slots out of order, as after an eviction
        c.tpos = np.stack([rng.permutation(cap) for _ in range(rows)]).astype(np.int32)
    c.forget_past(lens)
    kv, ld = c.put(), dev(np.asarray(lens, np.int32))
    m = torch.full((rows, budget), -9, dtype=torch.int32, device="cuda")
    after = ld if in_place else torch.zeros_like(ld)
    ao = None if in_place else torch.full((rows, budget + 2), 5.0, device="cuda")
    to = None if in_place else torch.full((rows, budget + 2), 5, dtype=torch.int32, device="cuda")
    D.kv_evict_q8(kv, ld, budget, sink, recent, m, after, acc_out=ao, tpos_out=to)
    assert after.tolist() == [min(n, budget) for n in lens]
    plans = [evict_plan(c.acc[b], c.tpos[b], n, budget, sink, recent) for b, n in enumerate(lens)]
    assert m.cpu().numpy().tolist() == plans
    aw, tw = np.full((rows, budget + 2), 5.0, np.float32), np.full((rows, budget + 2), 5, np.int32)
    for b, plan in enumerate(plans):
        for x, s in enumerate(plan):
            if s >= 0:
                aw[b, x], tw[b, x] = c.acc[b, s], c.tpos[b, s]
                for a in (c.k, c.v, c.ks, c.vs) + ((c.acc, c.tpos) if in_place else ()):
                    a[b, x] = a[b, s]
    c.same_as_device()
    if not in_place:
        assert np.array_equal(ao.cpu().numpy().view(np.uint32), aw.view(np.uint32))
        assert np.array_equal(to.cpu().numpy(), tw)


@gpu
def test_eviction_without_positions_takes_the_slot_for_the_position():
    rng = np.random.default_rng(3)
    c = Cache(rng, 1, 100, 1, 64)
    kv = c.put()
    bare = D.KvCache(c.d["kc"], c.d["ks"], c.d["vt"], c.d["vs"], 1, 64, acc=c.d["acc"])
    ld = dev(np.array([100], np.int32))
    m, after = torch.zeros(1, 60, dtype=torch.int32, device="cuda"), torch.zeros_like(ld)
    to = torch.zeros(1, 60, dtype=torch.int32, device="cuda")
    D.kv_evict_q8(bare, ld, 60, 4, 10, m, after, tpos_out=to)
    want = evict_plan(c.acc[0], c.tpos[0], 100, 60, 4, 10)
    assert m[0].tolist() == want and to[0].tolist() == want
    assert np.array_equal(c.d["acc"][0, :60].cpu().numpy(), c.acc[0, want])
    del kv


@gpu
@pytest.mark.parametrize("ring", [0, 40])
def test_tree_rows_enter_the_cache_as_single_rows_do(ring):
    """qkv_post_tree against qkv_post, whose slot is the row's position."""
    rng = np.random.default_rng(ring)
    rows, T, H, kvh, hd = 2, 5, 4, 2, 64
    lens = np.array([50, 37], np.int32)
    cap = 44 if ring else 60
    c = Cache(rng, rows, cap, kvh, hd, ring)
    kv = c.put()
    _, _, depth = random_tree(rng, rows, T)
    pos = (lens[:, None] + depth).astype(np.int32).reshape(-1)
    q, k, v = (rng.standard_normal((rows * T, h * hd)).astype(np.float32) for h in (H, kvh, kvh))
    qn, kn = (rng.uniform(0.5, 1.5, hd).astype(np.float32) for _ in range(2))
    inv = (1.0 / 10000.0 ** (np.arange(0, hd, 2) / hd)).astype(np.float32)
    cs = dev(D.rope_table(64, hd, inv))
    a = [dev(x) for x in (q, k, v)]
    D.qkv_post_tree(kv, *a, H, T, dev(qn), dev(kn), 1e-6, dev(inv), dev(pos), dev(lens), cs=cs)
    # one cache per row, the slot being the position
    each = Cache(rng, rows * T, 64, kvh, hd)
    each.put()
    d = each.d
    w = [dev(x) for x in (q, k, v)]
    D.qkv_post(*w, rows * T, H, kvh, hd, dev(qn), dev(kn), 1e-6, dev(inv), dev(pos), 0, 64,
               d["kc"], d["kc"].stride(0), d["ks"], d["ks"].stride(0), d["vt"], d["vt"].stride(0),
               d["vs"], d["vs"].stride(0), cs=cs)
    assert all(torch.equal(x, y) for x, y in zip(a, w))
    k1, s1, v1 = d["kc"].cpu().numpy(), d["ks"].cpu().numpy(), d["vs"].cpu().numpy()
    vt = d["vt"].cpu().numpy().reshape(rows * T, 16, kvh * hd, 4)
    for b in range(rows):
        for i in range(T):
            r, p = b * T + i, pos[b * T + i]
            s = (lens[b] + i) % ring if ring else lens[b] + i
            c.k[b, s], c.v[b, s] = k1[r, p], vt[r, p // 4, :, p % 4]
            c.ks[b, s], c.vs[b, s], c.tpos[b, s] = s1[r, p], v1[r, p], p
    c.same_as_device()


# ------------------------------------------------------- streams and graphs
@gpu
def test_on_another_stream_and_in_a_graph():
    rng = np.random.default_rng(13)
    lens, T, H, kvh, hd = [400, 222], 6, 8, 2, 128
    cache, q, mask, pos = setup(rng, lens, T, H, kvh, hd)
    kv, qd, ld, w, pd, out, lse = run_attend(cache, q, H, T, lens, mask, pos, 0)
    D.attend_accum_q8(qd, kv, H, T, ld, lse, mask=w, pos=pd, decay=0.5)
    acc = cache.d["acc"].clone()
    kv = cache.put()
    side = torch.cuda.Stream()
    out2, lse2 = torch.zeros_like(out), torch.zeros_like(lse)
    ws = D.attend_workspace(kv, H, T)
    torch.cuda.synchronize()

    def step(stream=None, ws=None):
        D.attend_tree_q8(out2, qd, kv, H, T, ld, mask=w, pos=pd, lse=lse2, ws=ws, stream=stream)
        D.attend_accum_q8(qd, kv, H, T, ld, lse2, mask=w, pos=pd, decay=0.5, ws=ws, stream=stream)

    step(side)
    side.synchronize()
    assert torch.equal(out2, out) and torch.equal(lse2, lse) and torch.equal(cache.d["acc"], acc)
    cache.d["acc"].copy_(dev(cache.acc))
    out2.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(ws=ws)
    out2.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out2, out) and torch.equal(cache.d["acc"], acc)


# ----------------------------------------------------------------- refusals
FAKE = 0x10000  # never dereferenced: every case fails on the host


def view(**kw):
    v = D.KvCache.__new__(D.KvCache)
    C.Structure.__init__(v)
    d = dict(kc=FAKE, ks=FAKE, vt=FAKE, vs=FAKE, acc=FAKE, tpos=FAKE, kc_stride=64 * 128,
             vt_stride=64 * 128, ks_stride=64, vs_stride=64, acc_stride=64, tpos_stride=64, rows=2,
             kv_heads=2, head_dim=64, cap=64, ring=0)
    d.update(kw)
    for k, x in d.items():
        setattr(v, k, x)
    return v


def err():
    return _lib.lib().fgm_cuda_last_error().decode()


BAD_VIEWS = [(dict(head_dim=96), "head_dim"), (dict(head_dim=576), "head_dim"),
             (dict(kv_heads=0), "kv_heads"), (dict(rows=-1), "rows"), (dict(cap=0), "cap"),
             (dict(ring=65), "ring"), (dict(kc=FAKE + 4), "aligned"), (dict(vt_stride=8200), "align"),
             (dict(kc_stride=64 * 128 - 16), "strides"), (dict(acc_stride=63), "strides"),
             (dict(vs_stride=63), "strides"), (dict(ks=None), "null"), (dict(ks=FAKE + 2), "4-byte")]


@pytest.mark.parametrize("kw,frag", BAD_VIEWS)
def test_caches_out_of_contract(kw, frag):
    L, v = _lib.lib(), view(**kw)
    p = C.byref(v)
    ws = 1 << 40
    assert L.fgm_cuda_attend_tree_q8(p, FAKE, 512, 4, 2, FAKE, None, None, 0, FAKE, 512, None, 0, 0,
                                     FAKE, ws, None) == -1 and frag in err()
    assert L.fgm_cuda_attend_accum_q8(p, FAKE, 512, 4, 2, FAKE, None, None, 0, FAKE, 4, 1, None, 1.0,
                                      FAKE, ws, None) == -1 and frag in err()
    assert L.fgm_cuda_attend_acc_q8(p, FAKE, 512, 4, FAKE, 1.0, FAKE, 512, FAKE, ws, None) == -1
    assert frag in err() or "ring" in err()
    assert L.fgm_cuda_kv_accept(p, 1, 2, FAKE, FAKE, FAKE, None, None) == -1 and frag in err()
    assert L.fgm_cuda_kv_evict_q8(p, FAKE, 8, 1, 1, FAKE, FAKE, None, None, 0, None) == -1
    assert frag in err()
    assert L.fgm_cuda_attend_workspace(p, 4, 2) == 0 and frag in err()


@pytest.mark.parametrize("kw,frag", [
    (dict(T=0), "T=0"), (dict(T=257), "T=257"), (dict(T=65), "cap"), (dict(heads=3), "heads"),
    (dict(heads=34), "heads"), (dict(q_ld=252), "q_ld"), (dict(q_ld=257), "q_ld"),
    (dict(out_ld=128), "out_ld"), (dict(window=-1), "window"), (dict(q=FAKE + 4), "aligned"),
    (dict(out=FAKE + 8), "aligned"), (dict(ws=FAKE + 16), "256-byte"), (dict(ws_bytes=0), "ws_bytes"),
    (dict(q=None), "null"), (dict(lens=None), "null"), (dict(ws=None), "null"),
    (dict(mask=FAKE + 4), "mask"), (dict(ring=32), "ring"), (dict(ring=32, window=32), "ring")])
def test_attention_out_of_contract(kw, frag):
    a = dict(T=2, heads=4, q_ld=256, out_ld=256, window=0, q=FAKE, out=FAKE, ws=FAKE,
             ws_bytes=1 << 40, lens=FAKE, mask=None, ring=0)
    a.update(kw)
    v = view(ring=a["ring"])
    L = _lib.lib()
    rc = L.fgm_cuda_attend_tree_q8(C.byref(v), a["q"], a["q_ld"], a["heads"], a["T"], a["lens"],
                                   a["mask"], None, a["window"], a["out"], a["out_ld"], None,
                                   0, 0, a["ws"], a["ws_bytes"], None)
    assert rc == -1 and frag in err(), err()
    if "out" in kw or "out_ld" in kw:
        return
    rc = L.fgm_cuda_attend_accum_q8(C.byref(v), a["q"], a["q_ld"], a["heads"], a["T"], a["lens"],
                                    a["mask"], None, a["window"], FAKE, 4, 1, None, 1.0,
                                    a["ws"], a["ws_bytes"], None)
    assert rc == -1 and frag in err(), err()


def test_other_refusals():
    L, v = _lib.lib(), view()
    p, ws = C.byref(v), 1 << 40
    bare = view(acc=None)
    assert L.fgm_cuda_attend_accum_q8(C.byref(bare), FAKE, 256, 4, 2, FAKE, None, None, 0, FAKE, 4, 1,
                                      None, 1.0, FAKE, ws, None) == -1 and "acc" in err()
    assert L.fgm_cuda_attend_accum_q8(p, FAKE, 256, 4, 2, FAKE, None, None, 0, None, 4, 1, None, 1.0,
                                      FAKE, ws, None) == -1 and "lse" in err()
    assert L.fgm_cuda_attend_acc_q8(C.byref(bare), FAKE, 256, 4, FAKE, 1.0, FAKE, 256, FAKE, ws,
                                    None) == -1 and "acc" in err()
    r = view(ring=64)
    assert L.fgm_cuda_attend_acc_q8(C.byref(r), FAKE, 256, 4, FAKE, 1.0, FAKE, 256, FAKE, ws,
                                    None) == -1 and "ring" in err()
    evict = lambda q, *a: L.fgm_cuda_kv_evict_q8(q, FAKE, *a)  # noqa: E731
    assert evict(C.byref(r), 8, 1, 1, FAKE, FAKE, None, None, 0, None) == -1 and "ring" in err()
    assert evict(p, 0, 1, 1, FAKE, FAKE, None, None, 0, None) == -1 and "budget" in err()
    assert evict(p, 65, 1, 1, FAKE, FAKE, None, None, 0, None) == -1 and "budget" in err()
    assert evict(p, 8, -1, 1, FAKE, FAKE, None, None, 0, None) == -1 and "sink" in err()
    assert evict(p, 8, 1, 1, FAKE, FAKE, FAKE, None, 7, None) == -1 and "out_stride" in err()
    assert evict(p, 8, 1, 1, None, FAKE, None, None, 0, None) == -1 and "null" in err()
    assert evict(C.byref(bare), 8, 1, 1, FAKE, FAKE, None, None, 0, None) == -1 and "acc" in err()
    big = view(rows=1, cap=524289)
    assert evict(C.byref(big), 8, 1, 1, FAKE, FAKE, None, None, 0, None) == -1 and "cap" in err()
    verify = L.fgm_cuda_tree_verify
    assert verify(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1, 0, None) == -1 and "T=0" in err()
    assert verify(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1, 257, None) == -1 and "T=257" in err()
    assert verify(FAKE, FAKE, None, FAKE, FAKE, FAKE, 1, 4, None) == -1 and "null" in err()
    assert L.fgm_cuda_tree_mask(FAKE, FAKE, FAKE, None, 1, 4, None) == -1 and "null" in err()
    assert L.fgm_cuda_tree_mask(FAKE, None, FAKE, None, 1, 257, None) == -1 and "T=257" in err()
    assert L.fgm_cuda_tree_mask(FAKE + 4, None, FAKE, None, 1, 4, None) == -1 and "8-byte" in err()
    assert L.fgm_cuda_kv_accept(p, 1, 65, FAKE, FAKE, FAKE, None, None) == -1 and "T=65" in err()
    assert L.fgm_cuda_kv_accept(p, 1, 2, FAKE, FAKE, FAKE, FAKE, None) == -1 and "lens_new" in err()
    two = (D.KvCache * 2)(view(), view(rows=1))
    assert L.fgm_cuda_kv_accept(two, 2, 2, FAKE, FAKE, FAKE, None, None) == -1 and "layer 1" in err()
    post = lambda q, T, **k: L.fgm_cuda_qkv_post_tree(  # noqa: E731
        q, FAKE, k.get("q_ld", 256), FAKE, FAKE, 128, 4, T, FAKE, FAKE, 1e-6, FAKE, None,
        k.get("positions", 0), FAKE, FAKE, None)
    assert post(p, 0) == -1 and "T=0" in err()
    assert post(p, 2, q_ld=255) == -1 and "q_ld" in err()
    assert post(p, 2, positions=4) == -1 and "rope" in err()
    assert post(C.byref(view(ring=3)), 4) == -1 and "ring" in err()


def test_empty_batches_need_no_device():
    L, v = _lib.lib(), view(rows=0)
    p = C.byref(v)
    assert L.fgm_cuda_attend_tree_q8(p, None, 256, 4, 2, None, None, None, 0, None, 256, None, 0, 0,
                                     None, 0, None) == 0
    assert L.fgm_cuda_attend_acc_q8(p, None, 256, 4, None, 1.0, None, 256, None, 0, None) == 0
    assert L.fgm_cuda_kv_evict_q8(p, None, 8, 1, 1, None, None, None, None, 0, None) == 0
    assert L.fgm_cuda_kv_accept(p, 1, 2, None, None, None, None, None) == 0
    assert L.fgm_cuda_tree_verify(None, None, None, None, None, None, 0, 4, None) == 0


def test_views_check_their_tensors():
    kc, s = torch.zeros(2, 8, 64, dtype=torch.int8), torch.zeros(2, 8)
    vt = torch.zeros(2, 512, dtype=torch.int8)
    D.KvCache(kc, s, vt, s, 1, 64)
    with pytest.raises(ValueError, match="kc"):
        D.KvCache(kc, s, vt, s, 2, 64)
    with pytest.raises(ValueError, match="ks"):
        D.KvCache(kc, s.double(), vt, s, 1, 64)
    with pytest.raises(ValueError, match="vt"):
        D.KvCache(kc, s, vt[:, :500], s, 1, 64)
    with pytest.raises(ValueError, match="vs"):
        D.KvCache(kc, s, vt, s[:1], 1, 64)
    with pytest.raises(ValueError, match="contiguous"):
        D.KvCache(kc, s, torch.zeros(2, 512, 2, dtype=torch.int8)[:, :, 0], s, 1, 64)
    with pytest.raises(ValueError, match="acc"):
        D.KvCache(kc, s, vt, s, 1, 64, acc=torch.zeros(2, 7))
    with pytest.raises(ValueError, match="mask has to be contiguous"):
        D._flat(lens=None, mask=torch.zeros(4, 4).t())
    with pytest.raises(ValueError, match="lens has to be contiguous torch.int32, not torch.int64"):
        D._flat(lens=torch.tensor([3, 4]))


# ------------------------------------------------------------- all together
@gpu
def test_speculative_decoding_gives_the_tokens_of_single_steps():
    """The example: the same greedy tokens in fewer steps, and a cache held to
    its budget goes on generating."""
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))
    import speculative_decode as S
    first = torch.tensor([3, 77], dtype=torch.int32, device="cuda")
    n = 48
    plain = S.generate(S.Model(2, n + 32), first, n).tolist()
    spec, steps = S.speculate(S.Model(2, n + 32), first, n, 8)
    assert [s[:n] for s in spec] == plain
    assert steps < n
    model = S.Model(2, 64)
    held, _ = S.speculate(model, first, n, 8, budget=24)
    assert all(len(h) >= n for h in held) and int(model.lens.max()) <= 24 + 8
    for kv in model.caches:  # the first tokens and the newest are still there
        tpos = kv._keep[5].cpu().numpy()
        for b, m in enumerate(model.lens.tolist()):
            assert set(range(4)) <= set(tpos[b, :m].tolist())
            assert len(set(tpos[b, :m].tolist())) == m
