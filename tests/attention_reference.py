"""A cache of keys and values in pages, appending and attention in 64 bits, for the tests.

Tolerance of attention, derived once (`Attention.bound`), in front of the one rounding of the result to its type.  With weights p_j (of sum 1),
entries v_j and A = sum_j p_j |v_j|:
  * a weight, its scale and an entry are rounded to at most 16 bits each on their way to a matrix instruction: three factors off by u each
    (u = 2^-11; 2^-8 where a cache of bf16 floats is multiplied as it is, weights and entries in bf16; nothing for f32): 3 u A, and the
    sums of weights and of products, n additions of f32 each: 2 n 2^-23 A where instructions may round towards zero;
  * a score off by d multiplies its weight by 1 + d, and the sum by at most as much: 2 d A.  d <= u_k B + (dim + 8) 2^-23 B with
    B = |scale| max_j sum_d |q_d k_jd|, u_k = 2 u (an entry of a key, an entry of a query, 16 bits each); the tanh adds cap 2^-20, the distance
    slope * distance * 2^-23, the exponential 2^-21 (|t| + |largest t| + 1) of itself.
What 16 bits of the weights cannot hold at all is below 2^-24 of the largest weight times the largest entry."""
import numpy as np
import torch

from cubek_amd import Cache, ComputeClient, ElemType, QuantScheme, Scores, TensorHandleRef, attention
from matmul_reference import PARAM, TORCH, check_rounded, random_weight, storage

h = TensorHandleRef.from_torch


def on_device(codes, scheme):
    return torch.from_numpy(codes.view(np.int32) if codes.dtype == np.uint32 else codes).cuda()


class Pool:
    """One of the stored tensors of a cache with what it holds in 64 bits: `entries` [pages, kv_heads, page_size, dim]."""

    def __init__(self, oracle, rng, shape, scheme, elem, size=1.0):
        if scheme is None:
            floats = torch.tensor(rng.normal(0, size, shape), dtype=torch.float32).to(TORCH[elem])
            self.stored, self.scales, self.entries = floats.cuda(), None, floats.double().numpy()
            return
        codes, scales = random_weight(rng, scheme, shape)
        scales = (scales.double() * (2.0 ** 2 if scheme.value.size_bits() == 8 else 2.0 ** 6) * size).to(PARAM[int(scheme.param)])
        one = torch.ones(scheme.scales_shape(shape), dtype=PARAM[int(scheme.param)])
        numbers = oracle.from_bits(oracle.dequantize(codes, shape, storage(one), ElemType.F32, scheme), ElemType.F32).reshape(shape)
        self.entries = numbers.astype(np.float64) * scales.double().repeat_interleave(shape[-1] // scales.shape[-1], -1).numpy()
        self.stored, self.scales = on_device(codes, scheme), scales.cuda()


def laid_out(t, order):
    """The same tensor with other strides: pages of [place][head] (`slots`), or with gaps between pages, heads and slots (`gaps`)."""
    if t is None or order == "heads":
        return t
    if order == "slots":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros([n + extra for n, extra in zip(t.shape, (0, 1, 2, 16 if t.shape[-1] >= 16 else 3))], dtype=t.dtype, device=t.device)
    view = wide[:, :-1, :-2, :t.shape[-1]]
    view.copy_(t)
    return view


class Attention:
    """Sequences of (new tokens, keys) over a cache of random entries."""

    def __init__(self, oracle, seed, sequences, heads, kv_heads, dim, page, elem, scheme=None, order="heads", spare=3, spread=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.sequences, self.elem, self.dim, self.group = sequences, elem, dim, heads // kv_heads
        need = [-(-length // page) for _, length in sequences]
        pages, width = sum(need) + spare, max(max(need), 1)
        shape = (pages, kv_heads, page, dim)
        self.k, self.v = Pool(oracle, rng, shape, scheme, elem, 1.0), Pool(oracle, rng, shape, scheme, elem, 1.0)
        free = rng.permutation(pages)
        self.table = np.full((len(sequences), width), -7, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = free[at:at + n]
            at += n
        self.tokens = sum(n for n, _ in sequences)
        self.offsets = np.concatenate([[0], np.cumsum([n for n, _ in sequences])]).astype(np.int32)
        self.lengths = np.array([n for _, n in sequences], np.int32)
        self.q = torch.tensor(rng.normal(0, spread, (self.tokens, heads, dim)), dtype=torch.float32).to(TORCH[elem])
        self.kept = [laid_out(t, order) for t in (self.k.stored, self.v.stored, self.k.scales, self.v.scales)]
        keys, values, key_scales, value_scales = (None if t is None else h(t) for t in self.kept)
        self.cache = Cache(keys, values, scheme, key_scales, value_scales)
        self.rounds = elem != ElemType.F32
        self.u = 0.0 if elem == ElemType.F32 else 2.0 ** -8 if scheme is None and elem == ElemType.BF16 else 2.0 ** -11

    def of_sequence(self, pool, s, head):
        length = self.sequences[s][1]
        page = pool.entries.shape[2]
        return pool.entries[self.table[s, :-(-length // page)], head].reshape(-1, self.dim)[:length]

    def want(self, scale=None, cap=0.0, window=0, slopes=None, prefix=None):
        """The results [tokens, heads, dim] and how far they may be off in front of their rounding."""
        scale = self.dim ** -0.5 if scale is None else scale
        q, heads = self.q.double().numpy(), self.q.shape[1]
        y, bound = np.zeros(q.shape), np.zeros(q.shape)
        for s, (n, length) in enumerate(self.sequences):
            a = self.offsets[s]
            i, j = np.arange(length - n, length)[:, None], np.arange(length)[None]
            seen = j <= i
            if prefix is not None:
                seen = seen | (j < prefix[s])
            if window:
                seen = seen & (i - j < window)
            some = seen.any(1)
            if n == 0 or length == 0:
                continue
            for head in range(heads):
                k, v = self.of_sequence(self.k, s, head // self.group), self.of_sequence(self.v, s, head // self.group)
                qs = q[a:a + n, head]
                t = scale * (qs @ k.T)
                b = abs(scale) * (np.abs(qs) @ np.abs(k).T)
                if cap:
                    t = cap * np.tanh(t / cap)
                away = np.abs(i - j)
                if slopes is not None:
                    t = t - slopes[head] * away
                t = np.where(seen, t, -np.inf)
                top = np.where(some, np.where(seen, t, -np.inf).max(1), 0.0)
                p = np.exp(t - top[:, None])
                p /= np.maximum(p.sum(1, keepdims=True), 1e-300)
                v = np.where(seen.any(0)[:, None], v, 0.0)  # unseen by all
                y[a:a + n, head] = p @ v
                size = p @ np.abs(v)
                steps = np.where(seen, np.abs(np.where(seen, t, 0.0)), 0.0).max(1) if length else 0.0
                d = (2 * self.u + (self.dim + 8) * 2.0 ** -23) * np.where(seen, b, 0.0).max(1) + cap * 2.0 ** -20 + 2.0 ** -21 * (2 * steps + 1)
                if slopes is not None:
                    d = d + abs(slopes[head]) * np.where(seen, away, 0).max(1) * 2.0 ** -23
                most = np.abs(np.where(seen.any(0)[:, None], v, 0.0)).max() if length else 0.0
                bound[a:a + n, head] = size * (3 * self.u + 2 * length * 2.0 ** -23 + 2 * d[:, None]) + most * 2.0 ** -24
        return y, bound

    def call(self, workspace=True, q=None, y=None, **scores):
        q = self.q.cuda() if q is None else q
        y = torch.full(tuple(self.q.shape), 77.0, dtype=self.q.dtype, device="cuda") if y is None else y
        ints = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (self.table, self.offsets, self.lengths)]
        hold = {}
        for name, dtype in (("slopes", torch.float32), ("prefix", torch.int32)):
            if scores.get(name) is not None:
                hold[name] = torch.tensor(np.asarray(scores[name]), dtype=dtype).cuda()
                scores[name] = h(hold[name])
        size = attention.workspace_bytes(self.cache, h(q), h(ints[0]), self.elem) if workspace else 0
        space = torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")
        attention.launch_ref(ComputeClient.current(), self.cache, h(q), h(y), *(h(t) for t in ints), self.elem, Scores(**scores),
                             workspace=space.data_ptr() if size else 0, workspace_size=size)
        torch.cuda.synchronize()
        return y

    def check(self, what="", workspace=True, **scores):
        want, bound = self.want(**scores)
        got = self.call(workspace, **scores).double().cpu().numpy()
        owned = np.zeros(self.tokens, bool)
        for s in range(len(self.sequences)):
            owned[self.offsets[s]:self.offsets[s + 1]] = True
        check_rounded(got[owned], want[owned], bound[owned], self.elem, what)
