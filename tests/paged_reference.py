"""Attention through a paged pool in 64 bits, with the error its kernels may make (test helper).

``attention64`` computes softmax(q k^T scale) v over the values a pool stands for, and beside each
output the bound

    |out - exact| <= half a bf16 step of the output
                     + A (u + 2 d + n 2^-23 + 2^-20),        A = sum_j w_j |v_j|,

where w are the softmax weights, u is the rounding of p before the second product (half a step: 2^-8
in bf16, 2^-11 in f16), d the largest error of a score (fp32 accumulation of 128 products, at most
2^-16 of the sum of their magnitudes, the two e4m3 parts of a query row, 2^-22 of its largest value, and
the rounding of the exponent's argument, 2^-22 of the score; it enters the weights and their sum, hence
twice), n the number of keys (each sum of n terms in fp32), and 2^-20 covers ex2.approx and the merge
of partial results.
"""

from __future__ import annotations

import torch

from miniserve_b200.attention import SeqChunk
from miniserve_b200.kv_pool import layer_as_slots

U_BF16, U_F16 = 2.0**-8, 2.0**-11
SCALE = 128**-0.5


def tree_mask(parents: list[int]) -> torch.Tensor:
    n = len(parents)
    m = torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        j = i if parents[i] != -2 else -1
        while j >= 0:
            m[i, j] = True
            j = parents[j]
    return m


def visible(c: SeqChunk) -> torch.Tensor:
    """[num_new, context] which keys each new token sees."""
    n, cached = c.num_new, c.num_cached
    at = torch.arange(cached + n)
    if c.parents is None:
        return at[None, :] <= cached + torch.arange(n)[:, None]
    m = tree_mask(c.parents)
    return torch.cat([m.any(1, keepdim=True).expand(n, cached), m], 1)


def attention64(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                chunks: list[SeqChunk], u: float, scale: float = SCALE
                ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(out fp64, bound fp64, covered rows); rows that see nothing are zero with bound zero."""
    ks, vs = layer_as_slots(k_cache), layer_as_slots(v_cache)
    t, heads, _ = q.shape
    out = torch.zeros(t, heads, 128, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    rows = []
    for c in chunks:
        tab = torch.tensor(c.block_table)
        p = torch.arange(c.context_len)
        slots = (tab[p // 16] * 16 + p % 16).to(q.device)
        vis = visible(c).to(q.device)
        lo, hi = c.flat_start, c.flat_start + c.num_new
        rows.extend(range(lo, hi))
        for h in range(heads):
            k, v = ks[slots, h // 2].double(), vs[slots, h // 2].double()
            x = q[lo:hi, h].double()
            for a in range(0, c.num_new, 256):
                xs, see = x[a : a + 256], vis[a : a + 256]
                # Keys a row does not see must not reach it, whatever they hold.
                s = (xs @ k.nan_to_num(0, 0, 0).T) * scale
                bad = ~torch.isfinite(k).all(1)
                s = torch.where(bad[None, :], torch.nan, s)
                s = torch.where(see, s, -torch.inf)
                dead = ~see.any(1)
                s[dead] = 0.0
                w = torch.softmax(s, -1)
                w = torch.where(see, w, 0.0)
                vz = v.nan_to_num(0, 0, 0)
                o = w @ vz
                special = ~torch.isfinite(v)
                if bool(special.any()):
                    for j in special.any(1).nonzero().flatten().tolist():
                        add = torch.where(special[j], v[j], 0.0)
                        o = o + torch.where(see[:, j : j + 1], w[:, j : j + 1] * add[None, :], 0.0)
                mag = w @ vz.abs()
                sums = (xs.abs() @ k.nan_to_num(0, 0, 0).abs().T) * scale
                top = xs.abs().amax(-1, keepdim=True) * k.nan_to_num(0, 0, 0).abs().sum(-1)[None, :]
                d = 2.0**-16 * sums + 2.0**-22 * top * scale + 2.0**-22 * s.abs()
                d = torch.where(see, d, 0.0).nan_to_num(0.0).amax(-1, keepdim=True)
                b = 2.0**-8 * o.abs() + mag * (u + 2 * d + c.context_len * 2.0**-23 + 2.0**-20)
                o[dead], b[dead] = 0.0, 0.0
                out[lo + a : lo + a + xs.shape[0], h] = o
                bound[lo + a : lo + a + xs.shape[0], h] = b
    return out, bound, torch.tensor(sorted(rows), device=q.device)


def assert_close(got: torch.Tensor, ref: torch.Tensor, bound: torch.Tensor,
                 rows: torch.Tensor) -> None:
    g, r, b = got[rows].double(), ref[rows], bound[rows]
    special = ~torch.isfinite(r)
    assert torch.equal(torch.isnan(g), torch.isnan(r)), "NaN in other places than the definition's"
    assert torch.equal(g[special & ~torch.isnan(r)], r[special & ~torch.isnan(r)])
    over = torch.where(special, 0.0, (g - r).abs() - b)
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"{worst:.3e} over the bound; error {(g - r).abs()[~special].max().item():.3e}"
