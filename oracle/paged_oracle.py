"""Plain 64-bit statements of the paged-cache operators and of rotary positions with several axes (CPU, loops)."""

import math

import torch


def rotary(x, positions, inv_freq, sections):
    """``x [B, H, T, D]`` turned; ``positions [A, B, T]``; in fp64."""
    R = len(inv_freq)
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    angle = torch.stack([positions[axis[d]].double() * float(inv_freq[d]) for d in range(R)], -1)[:, None]
    y = x.double().clone()
    a, b = x[..., :R].double(), x[..., R: 2 * R].double()
    y[..., :R] = a * angle.cos() - b * angle.sin()
    y[..., R: 2 * R] = b * angle.cos() + a * angle.sin()
    return y


def place(table, row, page, P):
    """(page, place in it) of a row of a sequence's table, or None."""
    if row < 0 or row // page >= len(table):
        return None
    at = int(table[row // page])
    return (at, row % page) if 0 <= at < P else None


def write(k, v, k_pages, v_pages, table, lens, new_lens=None, positions=None, weights=None, row_positions=None, k_scale=None, v_scale=None):
    """In place, on CPU tensors."""
    B, H, T, _ = k.shape
    P, _, page, _ = k_pages.shape
    capacity = table.shape[1] * page
    for b in range(B):
        n = T if new_lens is None else min(max(int(new_lens[b]), 0), T)
        for t in range(n):
            r = int(lens[b]) - n + t
            if not 0 <= r < capacity:
                continue
            if weights is not None:
                weights[b, :, r] = 0
            if row_positions is not None:
                row_positions[b, :, r] = r if positions is None else positions[b, t]
            at = place(table[b], r, page, P)
            if at is None:
                continue
            for x, pages, scale in ((k, k_pages, k_scale), (v, v_pages, v_scale)):
                row = x[b, :, t].float()
                if scale is not None:
                    s = (row.abs().amax(-1) * torch.tensor(1 / 448, dtype=torch.float32)).clamp_min(1e-12)
                    scale[at[0], :, at[1]] = s
                    pages.view(torch.uint8)[at[0], :, at[1]] = (row / s[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
                else:
                    pages[at[0], :, at[1]] = x[b, :, t]


def _rows(pages, page, head, row):
    if pages.dtype == torch.float8_e4m3fn:  # (indexing does not take 8-bit floats)
        return pages.view(torch.uint8)[page, head, row].view(torch.float8_e4m3fn).double()
    return pages[page, head, row].double()


def attend(q, k_pages, v_pages, table, lens, context_size=None, back=0, sm_scale=None, k_scale=None, v_scale=None):
    """``(o [B, H, D], lse [B, H], weights [B, H, capacity], spread)`` in fp64.  ``spread``: for tolerances, per head the largest
    ``sum |q_d k_d|`` of a row, and per output element the sum of ``p |v|``."""
    B, H, D = q.shape
    P, H_kv, page, _ = k_pages.shape
    capacity = table.shape[1] * page
    sm_scale = 1 / math.sqrt(D) if sm_scale is None else sm_scale
    o, lse = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, dtype=torch.float64)
    w = torch.zeros(B, H, capacity, dtype=torch.float64)
    dots, mass = torch.zeros(B, H, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    for b in range(B):
        n = min(max(int(lens[b]), 0), capacity)
        rows = [r for r in range(n) if (context_size is None or (n - 1) // context_size - r // context_size <= back)]
        rows = [(r, place(table[b], r, page, P)) for r in rows]
        rows = [(r, at) for r, at in rows if at is not None]
        if not rows:
            continue
        idx = torch.tensor([r for r, _ in rows])
        pg, ro = (torch.tensor([at[i] for _, at in rows]) for i in (0, 1))
        for h in range(H):
            g = h // (H // H_kv)
            k, v = _rows(k_pages, pg, g, ro), _rows(v_pages, pg, g, ro)
            if k_scale is not None:
                k, v = k * k_scale[pg, g, ro].double()[:, None], v * v_scale[pg, g, ro].double()[:, None]
            s = (k @ q[b, h].double()) * sm_scale
            p = s.softmax(0)
            o[b, h], lse[b, h], w[b, h, idx] = p @ v, s.logsumexp(0) / math.log(2), p
            dots[b, h] = ((k.abs() @ q[b, h].double().abs()) * abs(sm_scale)).max()
            mass[b, h] = p @ v.abs()
    return o, lse, w, (dots, mass)


def evict(k_pages, v_pages, table, lens, weights, row_positions, budget, recent, k_scale=None, v_scale=None):
    """In place, on CPU tensors."""
    P, H_kv, page, _ = k_pages.shape
    capacity = table.shape[1] * page
    for b in range(len(lens)):
        n = min(max(int(lens[b]), 0), capacity)
        lens[b] = min(max(int(lens[b]), 0), budget)
        if n <= budget:
            continue
        for h in range(H_kv):
            w, pos = weights[b, h, :n].tolist(), row_positions[b, h, :n].tolist()
            newest = max(pos)

            def rank(r):
                first = pos[r] > newest - recent
                return (not first, -pos[r] if first else w[r] != w[r], 0 if first or w[r] != w[r] else -w[r], r)

            # rows without a page hold nothing and places without one take nothing
            held = [r for r in range(n) if place(table[b], r, page, P) is not None]
            places = [r for r in held if r < budget]
            kept = sorted(held, key=rank)[:len(places)]
            src, dst = sorted(r for r in kept if r >= budget), sorted(set(places) - set(kept))
            assert len(src) == len(dst)
            for s, d in zip(src, dst):
                weights[b, h, d], row_positions[b, h, d] = weights[b, h, s], row_positions[b, h, s]
                sp, dp = place(table[b], s, page, P), place(table[b], d, page, P)
                for x in (k_pages, v_pages, k_scale, v_scale):
                    if x is not None:
                        x = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
                        x[dp[0], h, dp[1]] = x[sp[0], h, sp[1]]
