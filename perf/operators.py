"""Answering from a paged key/value cache, as measurable cases: rotary positions with several axes, the write of new
tokens into the cache, attention of one new token per sequence over it, and eviction by accumulated attention weight.

``run`` computes a case in its plain form, elementary torch operations in fp32, or, where ``own`` is true, through the
public entry points of ``kernels_b200.streaming_attention``.  Sizes are those of the repository's own cases and
benchmark (head counts 4 to 32, head dims 64 and 128, chunks of 128 and 256, contexts of 512 to 16 384 tokens), or generic.

Layouts: a cache is ``k_pages``, ``v_pages`` ``[P, H_kv, page, D]``; row ``r`` of sequence ``b`` lies in page
``page_table[b, r // page]`` at ``r % page``.  Table entries outside ``[0, P)`` hold nothing.  8-bit caches (e4m3) have one
fp32 scale per row and head, ``[P, H_kv, page]``.  ``weights`` and ``row_positions`` are ``[B, H_kv, M * page]``: per
cached row, the attention weight it has received and the position of its token.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f8": torch.float8_e4m3fn}
ELSIZE = {"f32": 4, "f16": 2, "bf16": 2, "f8": 1}
LOG2E = 1.4426950408889634


def listed():
    return [
        # rotary positions of one new token of every stream of a server: launches and host time are what it costs
        dict(name="rotary_step", op="rotary", train=False, dtype="bf16", B=64, H=32, H_kv=8, T=1, D=128, axes=3, far=1000000),
        # training step over video frames: three axes, head dim 64, an odd number of tokens, forward and backward
        dict(name="rotary_train", op="rotary", train=True, dtype="f16", B=8, H=16, H_kv=16, T=4095, D=64, axes=3, far=0),
        # a long prompt of several conversations with shared key/value heads
        dict(name="rotary_prompt", op="rotary", train=False, dtype="bf16", B=4, H=32, H_kv=8, T=8192, D=128, axes=1, far=4096),
        # the newest token of every stream goes into the cache
        dict(name="write_step", op="write", dtype="bf16", cache="bf16", B=64, H_kv=8, D=128, T=1, page=64, lo=300, hi=512),
        # prompts of ragged lengths go into an 8-bit cache
        dict(name="write_prompt", op="write", dtype="bf16", cache="f8", B=8, H_kv=8, D=128, T=8192, page=64, lo=4096, hi=8192),
        # a model kept in full precision, its first few hundred tokens: the smallest call
        dict(name="step_small", op="attend", dtype="f32", cache="f32", B=2, H=4, H_kv=4, D=64, page=16, lo=256, hi=511, c=0, back=0, weigh=False),
        # a streaming encoder's newest frame: the operator's own mask, every head with keys of its own
        dict(name="step_window", op="attend", dtype="f16", cache="f16", B=64, H=16, H_kv=16, D=64, page=32, lo=2048, hi=4096, c=128, back=4, weigh=False),
        # a full server: ragged contexts, shared key/value heads
        dict(name="step_batch", op="attend", dtype="bf16", cache="bf16", B=64, H=32, H_kv=8, D=128, page=64, lo=4096, hi=8192, c=0, back=0, weigh=False),
        # one conversation over a long document, 8-bit cache, an odd length: the work has to be split along the cache
        dict(name="step_long", op="attend", dtype="bf16", cache="f8", B=1, H=32, H_kv=8, D=128, page=128, lo=131001, hi=131001, c=0, back=0, weigh=False),
        # the same with the attention weights summed up for a later eviction
        dict(name="step_weights", op="attend", dtype="bf16", cache="bf16", B=16, H=32, H_kv=8, D=128, page=64, lo=8192, hi=16384, c=0, back=0, weigh=True),
        # a cache held at its budget: one row too many after every token
        dict(name="evict_step", op="evict", cache="bf16", B=32, H_kv=8, D=128, page=64, lo=2049, hi=2049, budget=2048, recent=256),
        # prompts cut down to a budget after their prefill
        dict(name="evict_prompt", op="evict", cache="bf16", B=16, H_kv=8, D=128, page=64, lo=6000, hi=16384, budget=4096, recent=512),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# what a drawn case may cost at most, in bytes of work(): a part of the listed cases' largest
_MOST_BYTES = {"rotary": 6.0e8, "write": 2.0e8, "attend": 1.2e9, "evict": 3.0e8}


def draw(rng: random.Random):
    for _ in range(1000):
        case = _draw_one(rng)
        rows = case.get("hi", 0) * case["B"] * case["H_kv"] * case["D"]
        if work(case)["bytes"] <= _MOST_BYTES[case["op"]] and rows <= 3.0e8:
            return case
    raise RuntimeError("no case within the ranges")


def _draw_one(rng: random.Random):
    op = rng.choice(["rotary", "write", "attend", "attend", "attend", "evict"])
    H, H_kv = rng.choice([(4, 4), (8, 8), (12, 4), (16, 16), (16, 2), (32, 8), (32, 4), (24, 8), (20, 1)])
    D = rng.choice([64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    B = _log_int(rng, 1, 128)
    if op == "rotary":
        train = rng.random() < 0.5
        return dict(op=op, train=train, dtype=dtype, B=B, H=H, H_kv=H_kv, T=_log_int(rng, 1, 16384), D=D, axes=rng.choice([1, 2, 3]),
                    far=rng.choice([0, 1000, 1000000]))
    cache = "f8" if dtype != "f32" and rng.random() < 0.3 else dtype
    page = rng.choice([8, 16, 32, 64, 128, 48])
    hi = _log_int(rng, 1, 65536)
    if op == "write":
        T = _log_int(rng, 1, min(hi, 16384))
        return dict(op=op, dtype=dtype, cache=cache, B=B, H_kv=H_kv, D=D, T=T, page=page, lo=max(T, hi // 2), hi=hi)
    lo = max(1, hi // rng.choice([1, 2, 8]))
    if op == "attend":
        c, back = (_log_int(rng, 10, 300), rng.randint(0, 8)) if rng.random() < 0.3 else (0, 0)
        return dict(op=op, dtype=dtype, cache=cache, B=B, H=H, H_kv=H_kv, D=D, page=page, lo=lo, hi=hi, c=c, back=back, weigh=rng.random() < 0.3)
    hi = max(hi, 16)
    budget = max(1, int(hi * rng.uniform(0.1, 1.0)))
    return dict(op=op, cache=cache, B=B, H_kv=H_kv, D=D, page=page, lo=max(1, hi // 2), hi=hi, budget=budget, recent=int(budget * rng.uniform(0.0, 0.5)))


def _lens(case):
    """The sequences' lengths, spread over the case's range: they belong to the case, their order to the seed."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    return [hi if B == 1 else lo + (hi - lo) * b // (B - 1) for b in range(B)]


def _new_lens(case):
    """Tokens that a ragged batch of prompts writes per sequence: all but the longest are padded."""
    B, T = case["B"], case["T"]
    return [T if b == 0 else T - (T // 2) * b // B for b in range(B)]


def _seen(case, length):
    """Rows that a new token (the sequence's last row) attends to."""
    if not case["c"]:
        return length
    first = max(0, (length - 1) // case["c"] - case["back"]) * case["c"]
    return length - first


def _sections(case):
    half, axes = case["D"] // 2, case["axes"]
    if axes == 1:
        return [half]
    rest = half - half // 4  # time takes a quarter of the frequencies, height and width share what is left
    return [half // 4, rest] if axes == 2 else [half // 4, rest // 2, rest - rest // 2]


def work(case):
    op, B, H_kv, D = case["op"], case["B"], case["H_kv"], case["D"]
    if op == "rotary":
        n = B * case["T"] * (case["H"] + H_kv) * D
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2.0 * n * ELSIZE[case["dtype"]] + 4 * case["axes"] * B * case["T"]), "flops": passes * 3.0 * n}
    row = D * ELSIZE[case["cache"]] + (4 if case["cache"] == "f8" else 0)  # bytes of one cached row of one head, keys or values
    if op == "write":
        n = sum(_new_lens(case)) * H_kv
        return {"bytes": 2.0 * n * (D * ELSIZE[case["dtype"]] + row) + 8.0 * n, "flops": (4.0 if case["cache"] == "f8" else 0.0) * n * D + 1}
    if op == "attend":
        n = sum(_seen(case, length) for length in _lens(case))
        b = 2.0 * n * H_kv * row + 2.0 * B * case["H"] * D * ELSIZE[case["dtype"]] + 4.0 * n / case["page"] + 4.0 * B * case["H"]
        return {"bytes": b + (8.0 * n * H_kv if case["weigh"] else 0.0), "flops": 4.0 * n * case["H"] * D}
    b = 0.0
    for length in _lens(case):
        kept, recent = min(length, case["budget"]), min(case["recent"], case["budget"])
        over = length - kept
        moved = (recent * over / length + (kept - recent) * over / max(1, length)) if over else 0
        b += H_kv * (8.0 * length + 8.0 * kept + 4.0 * moved * row)
    return {"bytes": b, "flops": float(sum(_lens(case))) * H_kv}


# ---- inputs --------------------------------------------------------------------------------------------------------


def _randn(gen, shape, dtype, scale=1.0):
    if dtype == torch.float8_e4m3fn:
        return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=gen).mul_(100.0).clamp_(-448.0, 448.0).to(dtype)
    x = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)
    return x.mul_(scale) if scale != 1.0 else x


def _cache(case, gen):
    """Pages of a server that has run for a while: handed out in any order, some free, stale rows behind every sequence."""
    B, H_kv, D, page = case["B"], case["H_kv"], case["D"], case["page"]
    order = torch.randperm(B, generator=gen, device="cuda")
    lens = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")[order]
    M = -(-case["hi"] // page)
    need = (lens.long() + page - 1) // page
    first = torch.cumsum(need, 0) - need
    total = sum(-(-n // page) for n in _lens(case))
    P = total + 4
    handed = torch.randperm(P, generator=gen, device="cuda")
    j = torch.arange(M, device="cuda")
    held = j[None] < need[:, None]
    table = torch.where(held, handed[(first[:, None] + j[None]).clamp_max(P - 1)], -1).to(torch.int32).contiguous()
    dtype = DTYPES[case["cache"]]
    s = dict(case=case, lens=lens, page_table=table, order=order)
    s["k_pages"], s["v_pages"] = (_randn(gen, (P, H_kv, page, D), dtype) for _ in range(2))
    s["k_scale"] = s["v_scale"] = None
    if case["cache"] == "f8":
        s["k_scale"], s["v_scale"] = (torch.rand((P, H_kv, page), generator=gen, device="cuda") * 0.01 + 0.005 for _ in range(2))
    return s


def _bookkeeping(case, gen):
    """Weights and positions of a cache whose rows earlier evictions have put out of order."""
    B, H_kv, L = case["B"], case["H_kv"], -(-case["hi"] // case["page"]) * case["page"]
    weights = torch.empty((B, H_kv, L), device="cuda").exponential_(generator=gen).pow_(2)
    positions = torch.rand((B, H_kv, L), generator=gen, device="cuda").argsort(-1).to(torch.int32)
    return weights, positions


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "rotary":
        B, T, D, dtype = case["B"], case["T"], case["D"], DTYPES[case["dtype"]]
        q, k = (_randn(gen, (B, h, T, D), dtype) for h in (case["H"], case["H_kv"]))
        sections = _sections(case)
        start = torch.randint(0, case["far"] + 1, (B, 1), generator=gen, device="cuda")
        at = torch.arange(T, device="cuda")[None]
        axes = [start + at] if case["axes"] == 1 else [start + at // 256, start + at // 16 % 16, start + at % 16][: case["axes"]]
        inv_freq = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64, device="cuda") / n) for n in sections])
        s = dict(case=case, q=q, k=k, positions=torch.stack(axes).to(torch.int32).contiguous(), inv_freq=inv_freq, sections=sections)
        if case["train"]:
            s["grads"] = [_randn(gen, x.shape, dtype) for x in (q, k)]
            q.requires_grad_(), k.requires_grad_()
        return s
    s = _cache(case, gen)
    if op == "write":
        B, H_kv, T, D = case["B"], case["H_kv"], case["T"], case["D"]
        s["k"], s["v"] = (_randn(gen, (B, H_kv, T, D), DTYPES[case["dtype"]]) for _ in range(2))
        new = torch.tensor(_new_lens(case), dtype=torch.int32, device="cuda")[s["order"]]
        s["new_lens"] = torch.minimum(new, s["lens"])
        s["weights"], s["row_positions"] = _bookkeeping(case, gen)
        s["positions"] = (torch.arange(T, device="cuda")[None] + torch.randint(0, 100000, (B, 1), generator=gen, device="cuda")).to(torch.int32)
    elif op == "attend":
        s["q"] = _randn(gen, (case["B"], case["H"], case["D"]), DTYPES[case["dtype"]], 2.0)
        s["weights"] = _bookkeeping(case, gen)[0] if case["weigh"] else None
    else:
        s["weights"], s["row_positions"] = _bookkeeping(case, gen)
        # the sums and lengths after an eviction go to buffers of their own, so that a pass can be repeated
        s["out"] = (torch.zeros_like(s["lens"]), torch.zeros_like(s["weights"]), torch.zeros_like(s["row_positions"]))
    return s


# ---- the framework's calls -----------------------------------------------------------------------------------------


def _own(s):
    from kernels_b200 import streaming_attention as sa

    case = s["case"]
    if case["op"] == "rotary":
        out = sa.rotary_embedding(s["q"], s["k"], s["positions"], s["inv_freq"], s["sections"])
        return [*out, *torch.autograd.grad(out, (s["q"], s["k"]), s["grads"])] if case["train"] else list(out)
    scales = dict(k_scale=s["k_scale"], v_scale=s["v_scale"])
    pages = (s["k_pages"], s["v_pages"], s["page_table"], s["lens"])
    if case["op"] == "write":
        sa.paged_cache_write(s["k"], s["v"], *pages, new_lens=s["new_lens"], positions=s["positions"], weights=s["weights"],
                             row_positions=s["row_positions"], **scales)
        return _written(s)
    if case["op"] == "attend":
        o, lse = sa.paged_attention(s["q"], *pages, context_size=case["c"] or None, back_contexts=case["back"], weights=s["weights"],
                                    return_lse=True, **scales)
        return dict(o=o, lse=lse, weights=s["weights"])
    sa.paged_cache_evict(*pages, s["weights"], s["row_positions"], case["budget"], case["recent"], out=s["out"], **scales)
    return _evicted(s)


def _written(s):
    return {n: s[n] for n in ("k_pages", "v_pages", "k_scale", "v_scale", "weights", "row_positions")}


def _evicted(s):
    lens, weights, row_positions = s["out"]
    return dict(k_pages=s["k_pages"], v_pages=s["v_pages"], k_scale=s["k_scale"], v_scale=s["v_scale"], lens=lens, weights=weights,
                row_positions=row_positions)


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _plain_rotate(x, cos, sin):
    xf = x.float()
    a, b = xf.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)


def _plain_rotary(s):
    # far positions lose their angle in 32 bits
    bands = zip(s["positions"].double(), s["inv_freq"].split(s["sections"]))
    angle = torch.cat([at[..., None] * freq for at, freq in bands], -1)
    cos, sin = (f(angle).float()[:, None] for f in (torch.cos, torch.sin))
    out = [_plain_rotate(s[n], cos, sin) for n in ("q", "k")]
    return out + list(torch.autograd.grad(out, (s["q"], s["k"]), s["grads"])) if s["case"]["train"] else out


def _plain_quantize(x):
    scale = (x.float().abs().amax(-1) / 448.0).clamp_min(1e-12)
    return (x.float() / scale[..., None]).to(torch.float8_e4m3fn), scale


def _bytes(x):
    """8-bit floats as bytes: indexing does not take them."""
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _plain_write(s):
    case, page = s["case"], s["case"]["page"]
    T, P = case["T"], s["k_pages"].shape[0]
    t = torch.arange(T, device=s["lens"].device)
    row = (s["lens"] - s["new_lens"]).long()[:, None] + t[None]
    live = (t[None] < s["new_lens"][:, None]) & (row >= 0) & (row < s["page_table"].shape[1] * page)
    at = s["page_table"].long().gather(1, (row // page).clamp(0, s["page_table"].shape[1] - 1))
    b, i = torch.nonzero(live, as_tuple=True)
    row, at = row[b, i], at[b, i]
    s["weights"][b, :, row] = 0.0
    s["row_positions"][b, :, row] = s["positions"][b, i][:, None]
    held = (at >= 0) & (at < P)
    b, i, row, at = b[held], i[held], row[held] % page, at[held]
    for name in ("k", "v"):
        x = s[name].transpose(1, 2)[b, i]
        if case["cache"] == "f8":
            x, scale = _plain_quantize(x)
            s[name + "_scale"][at, :, row] = scale
        _bytes(s[name + "_pages"])[at, :, row] = _bytes(x)
    return _written(s)


def _plain_rows(pages, scale, table):
    """The rows that the table names, ``[B, H_kv, M * page, D]`` in 32 bits."""
    x = pages[table] if pages.dtype != torch.float8_e4m3fn else pages.view(torch.uint8)[table].view(torch.float8_e4m3fn)
    x = x.float() if scale is None else x.float() * scale[table][..., None]
    B, M, H_kv, page, D = x.shape
    return x.transpose(1, 2).reshape(B, H_kv, M * page, D)


def _plain_seen(s):
    """Which rows the new token of every sequence attends to, ``[B, M * page]``."""
    case, table, lens = s["case"], s["page_table"], s["lens"].long()
    r = torch.arange(table.shape[1] * case["page"], device=table.device)
    seen = (r[None] < lens[:, None]) & ((table >= 0) & (table < s["k_pages"].shape[0])).repeat_interleave(case["page"], 1)
    if case["c"]:
        seen &= (lens[:, None] - 1) // case["c"] - r[None] // case["c"] <= case["back"]
    return seen


def _plain_attend(s):
    case, table = s["case"], s["page_table"].long().clamp(0, s["k_pages"].shape[0] - 1)
    B, H, D, H_kv = case["B"], case["H"], case["D"], case["H_kv"]
    seen = _plain_seen(s)[:, None, None]
    q = s["q"].float().view(B, H_kv, H // H_kv, D)
    score = q @ _plain_rows(s["k_pages"], s["k_scale"], table).transpose(-1, -2) / math.sqrt(D)
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    empty = total == 0
    w = p / torch.where(empty, 1.0, total)
    v = torch.where(seen[:, 0, 0, None, :, None], _plain_rows(s["v_pages"], s["v_scale"], table), 0.0)
    o = (w @ v).reshape(B, H, D).to(s["q"].dtype)
    lse = torch.where(empty, 0.0, top * LOG2E + torch.log2(torch.where(empty, 1.0, total))).reshape(B, H)
    if case["weigh"]:
        s["weights"] += w.sum(2)
    return dict(o=o, lse=lse, weights=s["weights"])


def _plain_evict(s):
    case, page = s["case"], s["case"]["page"]
    B, H_kv, L = s["weights"].shape
    M, P = s["page_table"].shape[1], s["k_pages"].shape[0]
    lens, weights, row_positions = s["out"]
    r = torch.arange(L, device=s["lens"].device)
    live = (r[None] < s["lens"][:, None])[:, None].expand(B, H_kv, L)
    # rows by rank: the newest first, then by weight, of equals the lower row; rows that hold nothing come last
    newest = torch.where(live, s["row_positions"], -1).amax(-1, keepdim=True).long()
    w = torch.where(s["row_positions"].long() > newest - case["recent"], math.inf, s["weights"])
    rank = torch.sort(torch.where(live, w, -1.0), dim=-1, descending=True, stable=True).indices.argsort(-1)
    kept = live & (rank < case["budget"])
    weights.copy_(torch.where(live & (r < case["budget"]), s["weights"], weights))
    row_positions.copy_(torch.where(live & (r < case["budget"]), s["row_positions"], row_positions))
    # the i-th kept row behind the budget fills the i-th place that came free before it
    inside = r < min(case["budget"], L)
    src, dst = (torch.where(m, r, L).sort(-1).values for m in (kept & ~inside, live & ~kept & inside))
    b, h, i = torch.nonzero((src < L) & (dst < L), as_tuple=True)
    src, dst = src[b, h, i], dst[b, h, i]
    weights[b, h, dst], row_positions[b, h, dst] = s["weights"][b, h, src], s["row_positions"][b, h, src]
    lens.copy_(s["lens"].clamp(0, case["budget"]))
    sp, dp = (s["page_table"].long()[b, (x // page).clamp_max(M - 1)] for x in (src, dst))
    ok = (sp >= 0) & (sp < P) & (dp >= 0) & (dp < P)
    h, sp, sr, dp, dr = h[ok], sp[ok], src[ok] % page, dp[ok], dst[ok] % page
    for x in (s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]):
        if x is not None:
            _bytes(x)[dp, h, dr] = _bytes(x)[sp, h, sr]
    return _evicted(s)


def run(s):
    if own:
        return _own(s)
    return dict(rotary=_plain_rotary, write=_plain_write, attend=_plain_attend, evict=_plain_evict)[s["case"]["op"]](s)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def _exact_rotary(s):
    out = []
    first = [sum(s["sections"][:a]) for a in range(len(s["sections"]))]
    parts = [s["positions"][a].double()[..., None] * s["inv_freq"][first[a]: first[a] + n] for a, n in enumerate(s["sections"])]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.cat(parts, -1))[:, None]
    tensors = [(s["q"], turn), (s["k"], turn)]
    if s["case"]["train"]:  # the gradient turns the other way
        tensors += [(g, turn.conj()) for g in s["grads"]]
    for x, by in tensors:
        half = x.shape[-1] // 2
        z = torch.complex(x.detach()[..., :half].double(), x.detach()[..., half:].double()) * by
        out.append(torch.cat([z.real, z.imag], -1))
    return out


def _exact_write(s):
    case, page, P = s["case"], s["case"]["page"], s["k_pages"].shape[0]
    got = {n: None if x is None else x.to(torch.float64) for n, x in _written(s).items() if n != "row_positions"}
    got["row_positions"] = s["row_positions"].clone()
    for b, (length, new) in enumerate(zip(s["lens"].tolist(), s["new_lens"].tolist())):
        rows = torch.arange(length - new, length, device="cuda")
        got["weights"][b, :, rows] = 0.0
        got["row_positions"][b, :, rows] = s["positions"][b, :new]
        at = s["page_table"][b].long()[rows // page]
        for name in ("k", "v"):
            x = s[name][b, :, :new].double()
            if case["cache"] == "f8":
                scale = (x.abs().amax(-1) / 448).clamp_min(1e-12)
                got[name + "_scale"][at, :, rows % page] = scale.T
                x = x / scale[..., None]
            got[name + "_pages"][at, :, rows % page] = x.transpose(0, 1)
    return got


def _exact_attend(s):
    case, page = s["case"], s["case"]["page"]
    B, H, D, H_kv = case["B"], case["H"], case["D"], case["H_kv"]
    o, lse = torch.zeros((B, H, D), dtype=torch.float64, device="cuda"), torch.zeros((B, H), dtype=torch.float64, device="cuda")
    weights = None if s["weights"] is None else s["weights"].double()
    for b, length in enumerate(s["lens"].tolist()):
        first = length - _seen(case, length)
        rows = torch.arange(first, length, device="cuda")
        at = s["page_table"][b].long()[rows // page]
        for g in range(H_kv):
            k, v = (_exact_rows(s, n, at, g, rows % page) for n in ("k", "v"))
            heads = slice(g * (H // H_kv), (g + 1) * (H // H_kv))
            score = s["q"][b, heads].double() @ k.T / math.sqrt(D)
            w = score.softmax(-1)
            o[b, heads] = w @ v
            lse[b, heads] = score.logsumexp(-1) / math.log(2)
            if weights is not None:
                weights[b, g, rows] += w.sum(0)
    return dict(o=o, lse=lse, weights=weights)


def _exact_rows(s, name, at, head, row):
    pages, scale = s[name + "_pages"], s[name + "_scale"]
    if scale is None:
        return pages[at, head, row].double()
    return pages.view(torch.uint8)[at, head, row].view(torch.float8_e4m3fn).double() * scale[at, head, row].double()[:, None]


def _exact_evict(s):
    case, page, budget = s["case"], s["case"]["page"], s["case"]["budget"]
    keep = {n: None if x is None else x.clone() for n, x in _evicted(s).items()}
    for b, length in enumerate(s["lens"].tolist()):
        keep["lens"][b] = min(length, budget)
        for h in range(case["H_kv"]):
            w, p = s["weights"][b, h, :length], s["row_positions"][b, h, :length]
            n = min(length, budget)
            keep["weights"][b, h, :n], keep["row_positions"][b, h, :n] = w[:n], p[:n]
            if length <= budget:
                continue
            recent = p > p.max() - case["recent"]
            # by weight, of equals the lower row first; then the newest before the others
            by_weight = torch.sort(w, descending=True, stable=True).indices
            order = torch.cat([by_weight[recent[by_weight]].sort().values, by_weight[~recent[by_weight]]])[:budget]
            src = order[order >= budget].sort().values
            free = torch.ones(budget, dtype=torch.bool, device="cuda")
            free[order[order < budget]] = False
            dst = free.nonzero()[:, 0]
            keep["weights"][b, h, dst], keep["row_positions"][b, h, dst] = w[src], p[src]
            at = s["page_table"][b].long()
            for name in ("k_pages", "v_pages", "k_scale", "v_scale"):
                if keep[name] is not None:
                    x = _bytes(keep[name])
                    x[at[dst // page], h, dst % page] = x[at[src // page], h, src % page]
    return {n: x.to(torch.float64) if x is not None and x.is_floating_point() else x for n, x in keep.items()}


def exact(case, seed):
    s = prepare(case, seed)
    return dict(rotary=_exact_rotary, write=_exact_write, attend=_exact_attend, evict=_exact_evict)[case["op"]](s)
