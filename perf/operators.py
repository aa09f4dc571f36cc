"""Cases of the paged-cache operators: the block-table plan, rotary positions with the append, and attention over the pages.

A step of a served model runs them in this order: the plan once, then for each layer the append and the attention.  Each
case is one call of one of the three, on buffers that a serving program holds.
"""
import functools
import math
import os
import sys

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one step of 64 utterances in flight (this engine's slot table), each bringing one frame
        dict(name="plan-decode-64", op="plan", requests=64, cached=594, arriving=1, page=16, mix=1),
        # a burst of admissions: 509 prompts of up to 512 rows on top of shared voices, pages of odd size
        dict(name="plan-burst-509", op="plan", requests=509, cached=125, arriving=512, page=24, mix=2),
        # the language model's decode step: 64 rows, 16 heads of 64, interleaved pairs, float rows filed as bf16
        dict(name="rotary-decode-64", op="rotary", rows=64, heads=16, kv_heads=16, dim=64, rot=64, interleaved=True, type="f32",
             cache="bf16", page=16, reach=600, mix=3),
        # an odd chunk at far positions: a third of the head rotated, halves layout, small pages
        dict(name="rotary-far-1001", op="rotary", rows=1001, heads=12, kv_heads=4, dim=96, rot=32, interleaved=False, type="f16",
             cache="f16", page=7, reach=1 << 20, mix=4),
        # a long prompt's chunk with grouped heads
        dict(name="rotary-chunk-8192", op="rotary", rows=8192, heads=32, kv_heads=8, dim=128, rot=128, interleaved=False, type="bf16",
             cache="bf16", page=64, reach=65536, mix=5),
        # first-chunk latency: a single stream of the float engine, one new row
        dict(name="attend-one-f32", op="attend", requests=1, new=1, context=218, heads=16, kv_heads=16, dim=64, type="f32", cache="f32",
             page=16, window=0, sinks=0, mix=6),
        # 64 utterances in flight, one new row each, the bf16 engine's cache
        dict(name="attend-decode-64", op="attend", requests=64, new=1, context=594, heads=16, kv_heads=16, dim=64, type="bf16",
             cache="bf16", page=16, window=0, sinks=0, mix=7),
        # long contexts with grouped heads, one new row each
        dict(name="attend-decode-long", op="attend", requests=16, new=1, context=16384, heads=32, kv_heads=8, dim=128, type="f16",
             cache="f16", page=64, window=0, sinks=0, mix=8),
        # endless streams: a window over a far context, the first rows (the voice) stay visible
        dict(name="attend-decode-sinks", op="attend", requests=24, new=1, context=40000, heads=16, kv_heads=16, dim=64, type="bf16",
             cache="bf16", page=32, window=1000, sinks=62, mix=9),
        # prompts and single rows in one batch, pages of odd size
        dict(name="attend-mixed-33", op="attend", requests=33, new=300, context=2500, heads=24, kv_heads=8, dim=64, type="f16",
             cache="f16", page=24, window=0, sinks=0, mix=10),
        # chunks of long prompts that see a window and the sinks
        dict(name="attend-chunk-sinks", op="attend", requests=6, new=700, context=9000, heads=16, kv_heads=4, dim=128, type="bf16",
             cache="bf16", page=16, window=2000, sinks=4, mix=11),
        # one chunk of a long prompt
        dict(name="attend-chunk-2048", op="attend", requests=1, new=2048, context=16384, heads=32, kv_heads=8, dim=128, type="bf16",
             cache="bf16", page=64, window=0, sinks=0, mix=12),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    page = rng.choice([1, 7, 8, 16, 24, 32, 64, 100, 128])
    mix = rng.randrange(1 << 30)
    what = rng.choice(["plan", "rotary", "rotary", "attend", "attend", "attend", "attend"])
    if what == "plan":
        requests = spread(1, 600)
        return dict(op="plan", requests=requests, cached=spread(1, 4000), arriving=spread(1, max(2, 200000 // requests)), page=page, mix=mix)
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 8) if g * kv_heads <= 32])
    dim = rng.choice([64, 64, 128, 128, 32, 80, 96])
    kind, cache = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16")])
    if what == "rotary":
        rot = rng.choice([dim, dim, dim // 2])
        return dict(op="rotary", rows=spread(1, 8192), heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, interleaved=rng.random() < 0.5,
                    type=kind, cache=cache, page=page, reach=spread(500, 1 << 20), mix=mix)
    requests, context = spread(1, 64), spread(1, 16384)
    context = min(context, 262144 // requests + 1)
    new = rng.choice([1, 1, spread(1, 2048)])
    # the largest listed case: 2048 rows x 16384 keys x 32 heads; the plain form's scores stay under that
    new = max(1, min(new, context, int(2048 * 16384 * 32 / (requests * context * heads))))
    if kind == "f32":
        new = max(1, new // 8)
    window, sinks = rng.choice([(0, 0), (0, 0), (spread(1, 2 * context), 0), (spread(1, context), spread(1, 64))])
    return dict(op="attend", requests=requests, new=new, context=context, heads=heads, kv_heads=kv_heads, dim=dim, type=kind, cache=cache,
                page=page, window=window, sinks=sinks, mix=mix)


def _lengths(case):
    """Ragged lengths of a case: (already cached, arriving) for each request."""
    g = np.random.default_rng(case["mix"])
    n = case["requests"]
    if case["op"] == "plan":
        cached = g.integers(0, case["cached"] + 1, n)
        arriving = np.full(n, 1) if case["arriving"] == 1 else g.integers(0, case["arriving"] + 1, n)
        return cached, arriving
    total = g.integers(max(1, case["context"] // 4), case["context"] + 1, n)
    total[0] = case["context"]
    arriving = np.minimum(total, g.integers(1, case["new"] + 1, n))
    arriving[0] = case["new"]
    if case["new"] > 1:
        arriving[g.random(n) < 0.4] = 1          # single rows among the chunks
        arriving[0] = case["new"]
    return total - arriving, arriving


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    host = np.random.default_rng(int(seed))

    def normal(*shape, dtype, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dtype)

    def ints(a):
        return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)

    page = case["page"]
    s = dict(case=case)
    if case["op"] == "plan":
        cached, arriving = _lengths(case)
        have, need = -(-cached // page), -(-(cached + arriving) // page)
        width = int(need.max()) + 3
        order = host.permutation(int(need.sum()) + 17)          # the pool's pages
        table = np.full((case["requests"], width), -1)
        k = int(have.sum())
        table[np.arange(width) < have[:, None]] = order[:k]
        rows = int(arriving.sum())
        s.update(cached=ints(cached), arriving=ints(arriving), table=ints(table), free=ints(order[k:]), slots=ints(np.zeros(rows)),
                 positions=ints(np.zeros(rows)), cu=ints(np.zeros(case["requests"] + 1)), kv_len=ints(np.zeros(case["requests"])),
                 counts=ints(np.zeros(4)))
        return s
    kind, kept, d = _TYPES[case["type"]], _TYPES[case["cache"]], case["dim"]
    heads, kv_heads = case["heads"], case["kv_heads"]
    if case["op"] == "rotary":
        rows = case["rows"]
        g = np.random.default_rng(case["mix"])
        pages = -(-rows // page) + 5
        kv = normal(rows, 2 * kv_heads, d, dtype=kind)                         # rows of one product: keys, then values
        base = torch.arange(case["rot"] // 2, device=dev, dtype=torch.float64)
        s.update(q=normal(rows, heads, d, dtype=kind), k=kv[:, :kv_heads], v=kv[:, kv_heads:],
                 positions=ints((g.integers(0, case["reach"] - min(rows, case["reach"] - 1)) + np.arange(rows)) % case["reach"]),
                 slots=ints(host.permutation(pages * page)[:rows]), freq=10000.0 ** (-2.0 * base / case["rot"]),
                 q_out=torch.zeros(rows, heads, d, device=dev, dtype=kind),
                 k_pages=normal(pages, page, kv_heads, d, dtype=kept), v_pages=normal(pages, page, kv_heads, d, dtype=kept))
        return s
    cached, arriving = _lengths(case)
    total = cached + arriving
    need = -(-total // page)
    pages = int(need.sum()) + 3
    order = host.permutation(pages)
    table = np.full((case["requests"], int(need.max())), -1)
    table[np.arange(table.shape[1]) < need[:, None]] = order[:int(need.sum())]
    rows = int(arriving.sum())
    s.update(q=normal(rows, heads, d, dtype=kind, scale=1.5), k_pages=normal(pages, page, kv_heads, d, dtype=kept),
             v_pages=normal(pages, page, kv_heads, d, dtype=kept), table=ints(table), cu=ints(np.concatenate([[0], np.cumsum(arriving)])),
             kv_len=ints(total), out=torch.zeros(rows, heads, d, device=dev, dtype=kind), lse=torch.zeros(rows, heads, device=dev),
             most=int(arriving.max()), longest=int(total.max()))
    return s


@functools.lru_cache(None)
def _ops():
    sys.path.insert(0, os.path.join(os.getcwd(), "pocket-tts.cpp_amd", "pyhost"))
    import ptts_paged
    return ptts_paged


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if op == "plan":
        if own:
            _ops().plan(s["cached"], s["arriving"], s["free"], s["table"], case["page"], slot_map=s["slots"], positions=s["positions"],
                        cu_rows=s["cu"], kv_len=s["kv_len"], counts=s["counts"])
            return s["table"], s["slots"], s["positions"], s["cu"], s["kv_len"], s["counts"]
        return _plain_plan(s, case["page"])
    if op == "rotary":
        if own:
            _ops().rotary_append(s["q"], s["k"], s["v"], s["positions"], s["freq"], interleaved=case["interleaved"], q_out=s["q_out"],
                                 slot_map=s["slots"], k_pages=s["k_pages"], v_pages=s["v_pages"])
            return s["q_out"], s["k_pages"], s["v_pages"]
        return _plain_rotary(s, case)
    if own:
        _ops().attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["kv_len"], window=case["window"], sinks=case["sinks"],
                         max_rows=s["most"], max_kv=s["longest"], out=s["out"], lse=s["lse"])
        return s["out"], s["lse"]
    return _plain_attention(s, case)


def _plain_plan(s, page):
    cached, arriving = s["cached"].long(), s["arriving"].long()
    n, width = s["table"].shape
    rows, n_free = s["slots"].numel(), s["free"].numel()
    have, end = (cached + page - 1) // page, cached + arriving
    need = (end + page - 1) // page - have
    cu = torch.cat([torch.zeros_like(cached[:1]), torch.cumsum(arriving, 0)])
    at = torch.cumsum(need, 0) - need
    col = torch.arange(width, device=cached.device)[None, :] - have[:, None]
    pick = at[:, None] + col
    new = torch.where(pick < n_free, s["free"].long()[pick.clamp(0, max(n_free - 1, 0))], -1)
    table = torch.where((col >= 0) & (col < need[:, None]), new, s["table"].long())
    r = torch.arange(rows, device=cached.device)
    i = torch.searchsorted(cu[1:], r, right=True).clamp(max=n - 1)
    pos = cached[i] + r - cu[i]
    of = table[i, (pos // page).clamp(max=width - 1)]
    slots = torch.where((of >= 0) & (pos // page < width), of * page + pos % page, -1)
    used = need.sum()
    counts = torch.stack([cu[-1], used.clamp(max=n_free), (used - n_free).clamp(min=0), torch.zeros_like(used)])
    live = r < cu[-1]
    slots, pos = torch.where(live, slots, s["slots"].long()), torch.where(live, pos, s["positions"].long())
    return tuple(x.int() for x in (table, slots, pos, cu, end, counts))


def _turn(x, angle, interleaved):
    rot = 2 * angle.shape[1]
    c, n = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = x.float()
    part, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    else:
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        part = torch.cat([a * c - b * n, b * c + a * n], -1)
    return torch.cat([part, rest], -1)


def _plain_rotary(s, case):
    angle = s["positions"].double()[:, None] * s["freq"][None, :]
    at = s["slots"].long()
    q = _turn(s["q"], angle, case["interleaved"]).to(s["q_out"].dtype)
    k_pages, v_pages = s["k_pages"], s["v_pages"]
    k_pages.flatten(0, 1)[at] = _turn(s["k"], angle, case["interleaved"]).to(k_pages.dtype)
    v_pages.flatten(0, 1)[at] = s["v"].float().to(v_pages.dtype)
    return q, k_pages, v_pages


def _plain_attention(s, case):
    heads, kv_heads, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    cu, kv_len = s["cu"].long(), s["kv_len"].long()
    n, rows, longest, most = kv_len.numel(), s["q"].shape[0], s["longest"], s["most"]
    j = torch.arange(longest, device=cu.device)
    of = s["table"].long()[:, j // page].clamp(min=0)
    live = j[None, :] < kv_len[:, None]
    keys = s["k_pages"][of, j % page].float() * live[:, :, None, None]          # [n, longest, kv_heads, d]
    values = s["v_pages"][of, j % page].float() * live[:, :, None, None]
    t = torch.arange(most, device=cu.device)
    row = (cu[:-1, None] + t[None, :]).clamp(max=rows - 1)
    q = s["q"][row].float().reshape(n, most, kv_heads, heads // kv_heads, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = torch.matmul(q * d ** -0.5, keys.permute(0, 2, 3, 1)).unflatten(2, (heads // kv_heads, most))
    pos = (kv_len - (cu[1:] - cu[:-1]))[:, None] + t[None, :]
    seen = (j[None, None, :] <= pos[:, :, None]) & live[:, None, :]
    if case["window"] > 0:
        seen = seen & ((j[None, None, :] > pos[:, :, None] - case["window"]) | (j < case["sinks"])[None, None, :])
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    weights = (scores - top).exp_()
    del scores
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.flatten(2, 3), values.permute(0, 2, 1, 3)).unflatten(2, (heads // kv_heads, most)) / total.clamp(min=1e-38)
    lse = (total.log() + top).squeeze(-1)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, most, heads, d)
    lse = lse.permute(0, 3, 1, 2).reshape(n, most, heads)
    r = torch.arange(rows, device=cu.device)
    i = torch.searchsorted(cu[1:], r, right=True)
    return out[i, r - cu[i]].to(s["out"].dtype), lse[i, r - cu[i]]


def exact(case, seed):
    s = prepare(case, seed)
    page = case["page"]
    if case["op"] == "plan":
        return None
    if case["op"] == "rotary":
        rot, half = case["rot"], case["rot"] // 2
        e = torch.exp(1j * (s["positions"].double()[:, None] * s["freq"]).to(torch.complex128))[:, None]
        q, k_pages, v_pages = s["q"].double(), s["k_pages"].double(), s["v_pages"].double()

        def turned(x):
            y = x.clone()
            a = x[..., 0:rot:2] if case["interleaved"] else x[..., :half]
            b = x[..., 1:rot:2] if case["interleaved"] else x[..., half:rot]
            z = torch.complex(a.contiguous(), b.contiguous()) * e
            if case["interleaved"]:
                y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
            else:
                y[..., :half], y[..., half:rot] = z.real, z.imag
            return y

        page_of, inside = s["slots"].long() // page, s["slots"].long() % page
        k_pages[page_of, inside] = turned(s["k"].double())
        v_pages[page_of, inside] = s["v"].double()
        return turned(q), k_pages, v_pages
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["dim"]
    group = heads // kv_heads
    cu, lens, table = s["cu"].tolist(), s["kv_len"].tolist(), s["table"].long()
    out = torch.zeros(s["q"].shape, device=s["q"].device, dtype=torch.float64)
    lse = torch.zeros(s["lse"].shape, device=s["q"].device, dtype=torch.float64)
    for i, length in enumerate(lens):
        used = table[i, :-(-length // page)]
        k = s["k_pages"][used].flatten(0, 1)[:length].double()
        v = s["v_pages"][used].flatten(0, 1)[:length].double()
        for first in range(cu[i], cu[i + 1], 256):
            last = min(first + 256, cu[i + 1])
            p = torch.arange(first, last, device=k.device)[:, None] - cu[i + 1] + length
            j = torch.arange(length, device=k.device)[None, :]
            hidden = j > p
            if case["window"] > 0:
                hidden |= (j <= p - case["window"]) & (j >= case["sinks"])
            for h in range(heads):
                logits = s["q"][first:last, h].double() @ k[:, h // group].T / math.sqrt(d)
                logits[hidden] = -math.inf
                lse[first:last, h] = torch.logsumexp(logits, 1)
                out[first:last, h] = torch.exp(logits - lse[first:last, h, None]) @ v[:, h // group]
    return out, lse


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] == "plan":
        cached, arriving = _lengths(case)
        rows, n = int(arriving.sum()), case["requests"]
        fresh = int((-(-(cached + arriving) // case["page"]) + (-cached // case["page"])).sum())
        return {"bytes": 4 * (2 * n + 2 * fresh + 2 * rows + 2 * n + 1), "flops": 0}
    q_bytes, kv_bytes = case["heads"] * case["dim"] * size[case["type"]], case["kv_heads"] * case["dim"]
    if case["op"] == "rotary":
        row = 2 * q_bytes + 2 * kv_bytes * (size[case["type"]] + size[case["cache"]]) + 8
        return {"bytes": case["rows"] * row + 8 * case["rot"] // 2, "flops": case["rows"] * (case["heads"] + case["kv_heads"]) * case["rot"] * 3}
    cached, arriving = _lengths(case)
    pairs = keys = 0
    for c, a in zip(cached.tolist(), arriving.tolist()):
        p = np.arange(c, c + a)
        if case["window"] > 0:
            low = np.maximum(p - case["window"] + 1, 0)
            pairs += int((p - low + 1 + np.minimum(low, case["sinks"])).sum())
            first = max(0, c - case["window"] + 1)
            keys += c + a - first + min(first, case["sinks"])
        else:
            pairs += int((p + 1).sum())
            keys += c + a
    rows = int(arriving.sum())
    pages = int((-(-(cached + arriving) // case["page"])).sum())
    return {"bytes": 2 * keys * kv_bytes * size[case["cache"]] + 2 * rows * q_bytes + 4 * rows * case["heads"] + 4 * (pages + 2 * case["requests"]),
            "flops": 4 * pairs * case["heads"] * case["dim"]}
