"""Speculative decoding over int8 KV caches that are held to a budget.

    python examples/speculative_decode.py [--tokens N] [--budget SLOTS]

A small random decoder (the layer structure of the reference's forward pass,
fgm-core/src/forward.rs:469-654, at toy sizes) generates greedily in two ways:
one token per step, and with drafted trees of which a step verifies up to T
nodes at once.  Both run on the library's entries alone; what a step of the
second does, per layer and sequence:

  qkv_post_tree    the nodes' K / V rows into the cache, behind the committed
  attend_tree_q8   every node over the cache and its ancestors, with its lse
  tree_verify      (once) the longest path whose tokens the model would choose
  attend_accum_q8  that path's attention weights, added to the slots'
  kv_accept        its rows moved behind the committed ones, in all layers
  kv_evict_q8      a cache past its budget gives up the slots that were
                   attended to least

The single-token steps use attend_acc_q8, attention and accumulation in one.
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from fastgemma_b200 import device as D  # noqa: E402
from fastgemma_b200 import fgm_format as F  # noqa: E402

H, NH, KVH, HD, FF, L, V, G, EPS = 512, 8, 2, 64, 1024, 2, 512, 64, 1e-6
QD, KVD = NH * HD, KVH * HD
QKV = QD + 2 * KVD


class Model:
    """Random weights and the buffers of up to 16 rows; one KvCache per layer."""

    def __init__(self, rows, cap, seed=0):
        rng = np.random.default_rng(seed)
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        norm = lambda n: dev(rng.uniform(0.5, 1.5, n).astype(np.float32))  # noqa: E731

        def weight(n, k):
            w, s = F.synth_q4g(n, k, G, int(rng.integers(1 << 30)))
            return dev(w), dev((s.astype(np.float32) * 0.3).astype(np.float16).view(np.uint16))

        self.layers = [dict(qkv=weight(QKV, H), o=weight(H, QD), gu=weight(2 * FF, H),
                            dn=weight(H, FF), pre=norm(H), post=norm(H), pre_ff=norm(H),
                            post_ff=norm(H), qn=norm(HD) * 0.3, kn=norm(HD)) for _ in range(L)]
        self.embed = dev(rng.standard_normal((V, H)).astype(np.float32))
        self.final, self.head = norm(H), weight(V, H)
        self.inv_freq = dev((1.0 / 10000.0 ** (np.arange(0, HD, 2) / HD)).astype(np.float32))
        self.rows, self.cap = rows, cap
        z = lambda *s, d=torch.float32: torch.zeros(*s, dtype=d, device="cuda")  # noqa: E731
        self.caches = [D.KvCache(z(rows, cap, KVD, d=torch.int8), z(rows, cap),
                                 z(rows, (cap + 3) // 4 * 4 * KVD, d=torch.int8), z(rows, cap),
                                 KVH, HD, acc=z(rows, cap), tpos=z(rows, cap, d=torch.int32))
                       for _ in range(L)]
        self.all = D.kv_layers(self.caches)
        # slots in use per sequence; eviction keeps the layers' counts equal
        self.lens = z(rows, d=torch.int32)
        self.qkv, self.attn = z(16, QKV), z(16, QD)
        self.proj, self.gu, self.logits = z(16, H), z(16, 2 * FF), z(16, V)
        self.q_kept = [z(16, QD) for _ in range(L)]     # of the last step, for the accumulation
        self.lse = [z(16, NH) for _ in range(L)]
        self.qs, self.pa = z(16), D.packed_a(16, max(H, QD, FF))
        self.ws = {}

    def _gemm(self, M, n, k, w, out):
        D.gemm_q4g(M, n, k, self.pa, self.qs, w[0], w[1], G, out)

    def step(self, tokens, pos, T, mask=None):
        """Logits [rows * T][V] of T tokens per sequence at the given positions."""
        M = self.rows * T
        h = self.embed[tokens.long()].contiguous()
        if T not in self.ws:
            self.ws[T] = D.attend_workspace(self.caches[0], NH, T)
        w_post, proj = None, None
        for i, (p, kv) in enumerate(zip(self.layers, self.caches)):
            D.norm_prep(h, proj, w_post, p["pre"], M, H, EPS, self.qs, self.pa)
            self._gemm(M, QKV, H, p["qkv"], self.qkv)
            q, k, v = self.qkv[:, :QD], self.qkv[:, QD:QD + KVD], self.qkv[:, QD + KVD:]
            D.qkv_post_tree(kv, q, k, v, NH, T, p["qn"], p["kn"], EPS, self.inv_freq, pos,
                            self.lens, q_ld=QKV, kv_ld=QKV)
            if T == 1:
                D.attend_acc_q8(self.attn, q, kv, NH, self.lens, ws=self.ws[T], q_ld=QKV)
            else:
                D.attend_tree_q8(self.attn, q, kv, NH, T, self.lens, mask=mask, lse=self.lse[i],
                                 ws=self.ws[T], q_ld=QKV)
                self.q_kept[i][:M].copy_(q[:M])
            D.prep_rows(self.attn, QD, self.qs, self.pa, M, QD, 0)
            self._gemm(M, H, QD, p["o"], self.proj)
            D.norm_prep(h, self.proj, p["post"], p["pre_ff"], M, H, EPS, self.qs, self.pa)
            self._gemm(M, 2 * FF, H, p["gu"], self.gu)
            D.gelu_mul_prep(self.gu, self.gu[:, FF:], M, FF, self.qs, self.pa, ld=2 * FF)
            self._gemm(M, H, FF, p["dn"], self.proj)
            w_post, proj = p["post_ff"], self.proj
        D.norm_prep(h, proj, w_post, self.final, M, H, EPS, self.qs, self.pa)
        self._gemm(M, V, H, self.head, self.logits)
        return self.logits[:M]

    def commit(self, T, mask, path, n_acc):
        """The accepted path's weights to the slots, its rows behind the committed ones."""
        take = torch.zeros(self.rows, T + 1, dtype=torch.uint8, device="cuda")
        take.scatter_(1, torch.where(path < 0, T, path).long(), 1)
        take = take[:, :T].contiguous()
        for kv, q, lse in zip(self.caches, self.q_kept, self.lse):
            D.attend_accum_q8(q, kv, NH, T, self.lens, lse, mask=mask, take=take, ws=self.ws[T])
        new = torch.empty_like(self.lens)
        D.kv_accept(self.all, T, self.lens, path, n_acc, new)
        self.lens = new

    def evict(self, budget, recent):
        """Every layer's cache back to its budget (each keeps its own slots)."""
        after = torch.empty_like(self.lens)
        for kv in self.caches:
            slots = torch.empty(self.rows, budget, dtype=torch.int32, device="cuda")
            D.kv_evict_q8(kv, self.lens, budget, 4, recent, slots, after)
        self.lens = after


def generate(model, first, n, budget=None):
    """One token per step: [rows][n] tokens."""
    tok, out = first.clone(), []
    for i in range(n):
        pos = torch.full((model.rows,), i, dtype=torch.int32, device="cuda")
        tok = model.step(tok, pos, 1).argmax(-1).to(torch.int32)
        model.lens += 1
        out.append(tok)
        if budget and i + 1 > budget:
            model.evict(budget, budget // 4)
    return torch.stack(out, 1)


def draft(known, roots, T):
    """Trees from what followed each token so far: the last and the one before
    it as children, breadth first; unknown successors are guessed as the token
    itself.  tokens and parents [rows][T]."""
    tokens, parents = np.zeros((len(roots), T), np.int32), np.full((len(roots), T), -1, np.int32)
    for b, root in enumerate(roots):
        tokens[b, 0], n, at = root, 1, 0
        while n < T:
            for t in (known[b].get(int(tokens[b, at])) or [int(tokens[b, at])])[:2]:
                if n < T:
                    tokens[b, n], parents[b, n], n = t, at, n + 1
            at += 1
    return tokens, parents


def speculate(model, first, n, T, budget=None):
    """The same with trees of T nodes: ([rows][>= n] tokens as lists, steps)."""
    rows = model.rows
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    out, known = [[] for _ in range(rows)], [{} for _ in range(rows)]
    root = first.cpu().numpy()
    mask = torch.empty(rows, T, (T + 63) // 64, dtype=torch.int64, device="cuda")
    path = torch.empty(rows, T, dtype=torch.int32, device="cuda")
    n_acc, nxt, done = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(3))
    steps = 0
    while min(len(o) for o in out) < n:
        tokens, parents = draft(known, root, T)
        tok, par = dev(tokens), dev(parents)
        pos = torch.empty(rows * T, dtype=torch.int32, device="cuda")
        D.tree_mask(mask, pos, par, done)  # positions count tokens, not slots
        target = model.step(tok.flatten(), pos, T, mask).argmax(-1).to(torch.int32)
        target = target.reshape(rows, T).contiguous()
        D.tree_verify(path, n_acc, nxt, par, tok, target)
        model.commit(T, mask, path, n_acc)
        done += n_acc
        steps += 1
        if budget and int(model.lens.max()) > budget:
            model.evict(budget, budget // 4)
        walk, kept, root = path.cpu().numpy(), n_acc.cpu().numpy(), nxt.cpu().numpy()
        for b in range(rows):  # the path's drafted tokens, then the model's own next one
            new = [int(tokens[b, walk[b, j]]) for j in range(1, kept[b])] + [int(root[b])]
            for a, c in zip([int(tokens[b, 0])] + new, new):
                known[b][a] = [c] + [t for t in known[b].get(a, []) if t != c][:1]
            out[b] += new
    return out, steps


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=96)
    ap.add_argument("--nodes", type=int, default=8)
    ap.add_argument("--budget", type=int, default=0, help="slots each cache keeps (0: all)")
    a = ap.parse_args()
    rows, cap = 2, a.tokens + 64
    first = torch.tensor([3, 77], dtype=torch.int32, device="cuda")
    plain = generate(Model(rows, cap), first, a.tokens, a.budget)
    spec, steps = speculate(Model(rows, cap), first, a.tokens, a.nodes, a.budget)
    same = [sum(x == y for x, y in zip(s, p)) for s, p in zip(spec, plain.tolist())]
    print(f"{a.tokens} tokens for each of {rows} sequences: {a.tokens} single-token steps, {steps} "
          f"steps of {a.nodes}-node trees; equal tokens {same}")


if __name__ == "__main__":
    main()
