"""Operators of a serving step over shared prefixes: what a program calls for each, over the sizes it meets.

Kinds of case, in the order of a step:
* ``tables``: page tables, positions and slot maps of the step's tokens, built on the GPU from the request lengths.
* ``rope``: rotary positions of q and k (both layouts, part of the head, scaled frequencies) and the append of k and v
  to the pages that the slot map names.
* ``shared``: decode attention of a batch whose rows share prefixes by groups, over paged contexts.
* ``logprobs``: log probabilities of given tokens, entropy and the most likely alternatives of each row of logits.

Sizes are fixed by the case alone; values come from the seed.
"""
from __future__ import annotations

import math
import random
import zlib

import numpy as np
import torch

own = False
DEVICE = "cuda"
PAGE = 16


# ------------------------------------------------------------------ cases ------
def listed() -> list[dict]:
    return [
        # one decode step of a full server: 128 rows, one new token each, a page now and then
        dict(name="tables decode b128", kind="tables", batch=128, lo=65, hi=8100, prompts=0, plo=0, phi=0),
        # admission: long prompts join a batch that goes on decoding
        dict(name="tables 24 prompts + 40 rows", kind="tables", batch=64, lo=30, hi=6000, prompts=24, plo=100,
             phi=2900),
        # the smallest step: one token of the float32 tiny model
        dict(name="rope tiny f32 1", kind="rope", tokens=1, heads=4, kv_heads=2, dim=64, rot=64, layout="interleaved",
             scaling="none", theta=10000.0, far=64, dtype="f32"),
        # a decode step of 32 sequences, interleaved pairs over the whole head
        dict(name="rope decode b32", kind="rope", tokens=32, heads=32, kv_heads=8, dim=128, rot=128,
             layout="interleaved", scaling="none", theta=500000.0, far=4096, dtype="f16"),
        # a chunk of a long-context prompt: halves, half of the head, frequencies scaled by bands, far positions
        dict(name="rope half 4093 far", kind="rope", tokens=4093, heads=28, kv_heads=4, dim=128, rot=64, layout="half",
             scaling="bands", theta=1000000.0, far=131072, dtype="f16"),
        # a few requests behind one system prompt
        dict(name="shared b4 prefix 500", kind="shared", heads=32, kv_heads=8, groups="4:500", lo=1, hi=40),
        # a full server: 128 sequences behind one 1024-token prefix, ragged suffixes
        dict(name="shared b128 prefix 1024", kind="shared", heads=28, kv_heads=4, groups="128:1024", lo=64, hi=7168),
        # several samples for each of a few prompts of their own lengths
        dict(name="shared 7 prompts sampled", kind="shared", heads=32, kv_heads=8,
             groups="8:700 8:3500 5:1777 16:2048 1:999 8:64 11:1200", lo=5, hi=300),
        # many questions about one long document
        dict(name="shared b64 prefix 16000", kind="shared", heads=32, kv_heads=8, groups="64:16000", lo=20, hi=600),
        # the alternatives of one token of the tiny model
        dict(name="logprobs 1x1024 top5", kind="logprobs", rows=1, vocab=1024, top=5, dtype="f32", pad=0),
        # a decode step that returns alternatives
        dict(name="logprobs 32x128256 top20", kind="logprobs", rows=32, vocab=128256, top=20, dtype="f32", pad=0),
        # the scores of a prompt's own tokens, logits in half precision in rows wider than the vocabulary
        dict(name="score 1021x152064 f16 top2", kind="logprobs", rows=1021, vocab=152064, top=2, dtype="f16", pad=64),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["tables", "rope", "rope", "shared", "shared", "shared", "logprobs", "logprobs"])
    if kind == "tables":
        batch = _log(rng, 1, 512)
        hi = _log(rng, 20, 8100)
        prompts = rng.choice([0, rng.randint(0, min(batch, 32))])
        return dict(kind=kind, batch=batch, lo=rng.randint(0, hi), hi=hi, prompts=prompts, plo=rng.randint(0, 64),
                    phi=_log(rng, 65, 2900))
    if kind == "rope":
        heads, kv_heads, dim = rng.choice([(32, 8, 128), (28, 4, 128), (4, 2, 64), (16, 8, 96), (8, 8, 80),
                                           (8, 1, 256)])
        rot = rng.choice([dim, dim, dim // 2, dim // 4])
        return dict(kind=kind, tokens=_log(rng, 1, 4096), heads=heads, kv_heads=kv_heads, dim=dim, rot=rot,
                    layout=rng.choice(["interleaved", "half"]), scaling=rng.choice(["none", "linear", "bands"]),
                    theta=rng.choice([10000.0, 500000.0, 1000000.0]), far=_log(rng, 64, 131072),
                    dtype=rng.choice(["f16", "f16", "f32"]))
    if kind == "shared":
        heads, kv_heads = rng.choice([(32, 8), (28, 4), (16, 8), (8, 8), (16, 1)])
        n = rng.choice([1, 1, 1, rng.randint(2, 9)])
        batch = _log(rng, n, 128)
        cuts = sorted(rng.sample(range(1, batch), n - 1)) if n > 1 else []
        sizes = [b - a for a, b in zip([0] + cuts, cuts + [batch])]
        room = 1800000 // kv_heads  # tokens that the pools hold
        hi = _log(rng, 2, min(8000, room * 3 // 4 // batch))
        top = min(16000, room // 4 // n, 1000000 // batch)
        groups = " ".join(f"{m}:{rng.choice([0, _log(rng, 16, top), _log(rng, 16, top)])}" for m in sizes)
        return dict(kind=kind, heads=heads, kv_heads=kv_heads, groups=groups, lo=rng.randint(1, hi), hi=hi)
    vocab = rng.choice([1024, 16384, 128256, 152064, _log(rng, 100, 152064)])
    return dict(kind=kind, rows=_log(rng, 1, max(1, 70000000 // vocab)) if rng.random() < 0.5 else _log(rng, 1, 128),
                vocab=vocab, top=rng.choice([0, 1, 5, 20, rng.randint(1, 64)]), dtype=rng.choice(["f32", "f32", "f16"]),
                pad=rng.choice([0, 0, 1, 64]))


def _spread(n: int, lo: int, hi: int, salt: int) -> list[int]:
    """n whole numbers spread evenly between lo and hi in an order of their own (fixed by the case)."""
    v = [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(n * 1000003 + lo * 1009 + hi * 31 + salt).shuffle(v)
    return v


# ------------------------------------------------------------------ values -----
def _gen(seed: int, *what) -> torch.Generator:
    g = torch.Generator(device=DEVICE)
    g.manual_seed((seed * 2654435761 + zlib.crc32(repr(what).encode())) & 0x7FFFFFFFFFFF)
    return g


def _randn(shape, seed: int, *what, dtype=torch.float32) -> torch.Tensor:
    return torch.randn(shape, generator=_gen(seed, *what), device=DEVICE, dtype=torch.float32).to(dtype)


def _i32(v) -> torch.Tensor:
    return torch.tensor(v, dtype=torch.int32, device=DEVICE)


def _dtype(case: dict) -> torch.dtype:
    return torch.float16 if case["dtype"] == "f16" else torch.float32


def _frequencies(case: dict) -> tuple[list[float], float]:
    """Angles per position of the rot/2 pairs and the factor on cos and sin.  "linear" divides every frequency by 4;
    "bands" keeps the fast ones (over 4 turns in 8192 positions), divides the slow ones (under 1 turn) by 8, passes
    from one to the other linearly in the number of turns, and scales cos and sin a little up."""
    half = case["rot"] // 2
    f = [case["theta"] ** (-2.0 * i / case["rot"]) for i in range(half)]
    if case["scaling"] == "linear":
        return [v / 4.0 for v in f], 1.0
    if case["scaling"] == "bands":
        out = []
        for v in f:
            keep = min(1.0, max(0.0, (8192.0 * v / (2.0 * math.pi) - 1.0) / 3.0))
            out.append(keep * v + (1.0 - keep) * v / 8.0)
        return out, 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def _groups(case: dict) -> tuple[list[int], list[int]]:
    """(rows, prefix tokens) of the groups of a ``shared`` case, written "rows:prefix rows:prefix ..."."""
    pairs = [g.split(":") for g in case["groups"].split()]
    return [int(r) for r, _ in pairs], [int(p) for _, p in pairs]


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(tokens held, new tokens) of the rows of a ``tables`` case: prompts hold none yet."""
    b, p = case["batch"], case["prompts"]
    held = _spread(b, case["lo"], case["hi"], 1)
    new = [1] * b
    if p:
        where = random.Random(b * 7919 + p).sample(range(b), p)
        for w, n in zip(where, _spread(p, case["plo"], case["phi"], 2)):
            held[w], new[w] = 0, n
    return held, new


def prepare(case: dict, seed: int) -> dict:
    kind = case["kind"]
    if kind == "tables":
        held, new = _lengths(case)
        width = -(-max(h + n for h, n in zip(held, new)) // PAGE)
        have = [-(-h // PAGE) for h in held]
        need = sum(-(-(h + n) // PAGE) - a for h, n, a in zip(held, new, have))
        spare = 37
        order = torch.randperm(sum(have) + need + spare, generator=_gen(seed, "pages"), device=DEVICE).to(torch.int32)
        counts = _i32(have)
        col = torch.arange(width, device=DEVICE)[None, :]
        at = (torch.cumsum(counts, 0) - counts)[:, None] + col
        table = torch.where(col < counts[:, None], order[torch.clamp(at, max=order.numel() - 1)], 0).to(torch.int32)
        return dict(case=case, table=table.contiguous(), lens=_i32(held), new=_i32(new), head=_i32([5]),
                    free=torch.cat([order[:5], order[sum(have):]]).contiguous(), tokens=sum(new) + 3)
    if kind == "rope":
        t, hq, hk, d, dt = case["tokens"], case["heads"], case["kv_heads"], case["dim"], _dtype(case)
        qkv = _randn((t, (hq + 2 * hk) * d), seed, "qkv", dtype=dt)
        q, k, v = qkv.split([hq * d, hk * d, hk * d], dim=1)
        pages = -(-t // PAGE) + 3
        slots = torch.randperm(pages * PAGE, generator=_gen(seed, "slots"), device=DEVICE)[:t]
        freq, factor = _frequencies(case)
        pos = torch.randint(0, case["far"], (t,), generator=_gen(seed, "pos"), device=DEVICE, dtype=torch.int32)
        return dict(case=case, q=q.unflatten(1, (hq, d)), k=k.unflatten(1, (hk, d)), v=v.unflatten(1, (hk, d)), pos=pos,
                    slots=slots, freq=torch.tensor(freq, dtype=torch.float64, device=DEVICE), factor=factor,
                    k_pool=torch.zeros((pages, hk, PAGE, d), dtype=dt, device=DEVICE),
                    v_pool=torch.zeros((pages, hk, PAGE, d), dtype=dt, device=DEVICE))
    if kind == "shared":
        hq, hk, d = case["heads"], case["kv_heads"], 128
        groups, prefixes = _groups(case)
        batch = sum(groups)
        suffix = _spread(batch, case["lo"], case["hi"], 3)
        rows, used, first, lens = [], 0, 0, []
        for n, prefix in zip(groups, prefixes):
            whole = prefix // PAGE  # the prefix's last page, where it ends inside one, is each row's own copy
            common = list(range(used, used + whole))
            used += whole
            for b in range(first, first + n):
                length = prefix + suffix[b]
                own_pages = -(-length // PAGE) - whole
                rows.append(common + list(range(used, used + own_pages)))
                used += own_pages
                lens.append(length)
            first += n
        width = max(len(r) for r in rows)
        order = torch.randperm(used, generator=_gen(seed, "pages"), device=DEVICE).to(torch.int32)
        table = order[torch.tensor([r + [0] * (width - len(r)) for r in rows], device=DEVICE)].contiguous()
        shared = [p // PAGE * PAGE for p in prefixes]
        state = dict(case=case, q=_randn((batch, hq, d), seed, "q", dtype=torch.float16),
                     k_pool=_randn((used, hk, PAGE, d), seed, "k", dtype=torch.float16),
                     v_pool=_randn((used, hk, PAGE, d), seed, "v", dtype=torch.float16), table=table, lens=_i32(lens),
                     host_lens=lens, group_rows=_i32(np.cumsum([0] + groups).tolist()),
                     prefix=_i32(shared), scale=1.0 / math.sqrt(d))
        if own:
            from cacheir_amd import kernels

            state["workspace"] = kernels.shared_attention_workspace(batch, len(shared), hq, hk, d, PAGE, width,
                                                                    torch.float16, DEVICE)
        return state
    rows, vocab = case["rows"], case["vocab"]
    # logits of a model: a wide bulk and a few likely tokens
    wide = _randn((rows, vocab + case["pad"]), seed, "logits") * 2.5
    likely = torch.randint(0, vocab, (rows, 12), generator=_gen(seed, "likely"), device=DEVICE)
    wide.scatter_add_(1, likely, 9.0 + 2.0 * _randn((rows, 12), seed, "peaks"))
    pick = torch.randint(0, 12, (rows, 1), generator=_gen(seed, "pick"), device=DEVICE)
    state = dict(case=case, logits=wide.to(_dtype(case))[:, :vocab], ids=likely.gather(1, pick).squeeze(1))
    if own:
        from cacheir_amd import kernels

        state["workspace"] = kernels.token_logprobs_workspace(rows, vocab, case["top"], DEVICE)
    return state


# ------------------------------------------------------------------ passes -----
def run(state: dict):
    kind = state["case"]["kind"]
    return (_OWN if own else _PLAIN)[kind](state)


def _own_tables(s: dict):
    from cacheir_amd import kernels

    t = kernels.extend_page_tables(s["table"], s["lens"], s["new"], s["free"], s["head"], page_size=PAGE,
                                   max_tokens=s["tokens"])
    return [s["table"], t.seq_lens, t.free_head, t.offsets, t.positions, t.slot_map, t.granted]


def _own_rope(s: dict):
    from cacheir_amd import kernels

    q = kernels.rope_append(s["q"], s["k"], s["v"], s["pos"], s["slots"], s["freq"], s["k_pool"], s["v_pool"],
                            layout=s["case"]["layout"], factor=s["factor"])
    return [q, s["k_pool"], s["v_pool"]]


def _own_shared(s: dict):
    from cacheir_amd import kernels

    return kernels.paged_decode_attention_shared(s["q"], s["k_pool"], s["v_pool"], s["table"], s["lens"],
                                                 s["group_rows"], s["prefix"], scale=s["scale"],
                                                 workspace=s["workspace"])


def _own_logprobs(s: dict):
    from cacheir_amd import kernels

    r = kernels.token_logprobs(s["logits"], s["ids"], s["case"]["top"], workspace=s["workspace"])
    return [r.logprobs, r.entropy, r.top_ids, r.top_logprobs]


def _plain_tables(s: dict):
    table, lens, new = s["table"], s["lens"].long(), s["new"].long()
    width, tokens = table.shape[1], s["tokens"]
    ends = torch.cumsum(new, 0)
    starts = ends - new
    have, want = (lens + PAGE - 1) // PAGE, (lens + new + PAGE - 1) // PAGE
    fits = (want <= width) & (ends <= tokens)
    need = torch.where(fits, want - have, 0)
    upto = torch.cumsum(need, 0)
    ok = fits & ((need == 0) | (upto <= s["free"].numel() - s["head"].long()))
    col = torch.arange(width, device=table.device)[None, :]
    fresh = (col >= have[:, None]) & (col < want[:, None]) & ok[:, None]
    at = s["head"].long() + (upto - need)[:, None] + col - have[:, None]
    table = torch.where(fresh, s["free"][torch.clamp(at, 0, s["free"].numel() - 1)], table)
    j = torch.arange(tokens, device=table.device)
    row = torch.clamp(torch.searchsorted(ends, j, right=True), max=lens.numel() - 1)
    live = j < ends[-1]
    pos = torch.where(live, lens[row] + j - starts[row], 0)
    page = table[row, torch.clamp(pos // PAGE, max=width - 1)].long()
    slot = torch.where(live & ok[row], page * PAGE + pos % PAGE, -1)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=table.device), ends])
    granted = torch.where(ok, new, 0)
    return [table, (lens + granted).int(), (s["head"] + torch.where(ok, need, 0).sum()).int(), offsets.int(), pos.int(),
            slot, granted.int()]


def _plain_rope(s: dict):
    c = s["case"]
    rot = c["rot"]
    turn = s["pos"].double()[:, None] * s["freq"][None, :]
    cos, sin = (torch.cos(turn) * s["factor"]).float()[:, None, :], (torch.sin(turn) * s["factor"]).float()[:, None, :]

    def rotate(x):
        y = x.float().clone()
        if c["layout"] == "interleaved":
            a, b = y[..., 0:rot:2].clone(), y[..., 1:rot:2].clone()
            y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
        else:
            a, b = y[..., : rot // 2].clone(), y[..., rot // 2: rot].clone()
            y[..., : rot // 2], y[..., rot // 2: rot] = a * cos - b * sin, a * sin + b * cos
        return y.to(x.dtype)

    page, off = s["slots"] // PAGE, s["slots"] % PAGE
    s["k_pool"][page, :, off] = rotate(s["k"])
    s["v_pool"][page, :, off] = s["v"]
    return [rotate(s["q"]), s["k_pool"], s["v_pool"]]


def _plain_shared(s: dict):
    batch, hq, d = s["q"].shape
    hk = s["k_pool"].shape[1]
    out = torch.empty_like(s["q"])
    for b, n in enumerate(s["host_lens"]):
        pages = s["table"][b, : -(-n // PAGE)].long()
        k = s["k_pool"][pages].permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :n].float()
        v = s["v_pool"][pages].permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :n].float()
        q = s["q"][b].float().reshape(hk, hq // hk, d)
        w = torch.matmul(k, q.transpose(1, 2).contiguous()) * s["scale"]  # [kv head, token, query head]
        w = torch.exp(w - w.amax(dim=1, keepdim=True))
        o = torch.matmul(w.transpose(1, 2).contiguous(), v) / w.sum(dim=1)[:, :, None]
        out[b] = o.reshape(hq, d).to(out.dtype)
    return out


def _plain_logprobs(s: dict):
    x = s["logits"].float()
    d = x - x.amax(dim=1, keepdim=True)
    e = torch.exp(d)
    z = e.sum(dim=1, keepdim=True)
    logz = torch.log(z)
    entropy = logz - (e * d).sum(dim=1, keepdim=True) / z
    lp = d.gather(1, s["ids"][:, None]) - logz
    top = torch.sort(d, dim=1, descending=True, stable=True).indices[:, : s["case"]["top"]].contiguous()
    return [lp.squeeze(1), entropy.squeeze(1), top, d.gather(1, top) - logz]


_OWN = dict(tables=_own_tables, rope=_own_rope, shared=_own_shared, logprobs=_own_logprobs)
_PLAIN = dict(tables=_plain_tables, rope=_plain_rope, shared=_plain_shared, logprobs=_plain_logprobs)


# -------------------------------------------------------------- references -----
def exact(case: dict, seed: int):
    """What ``run`` returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    return dict(tables=_exact_tables, rope=_exact_rope, shared=_exact_shared, logprobs=_exact_logprobs)[case["kind"]](s)


def _exact_tables(s: dict):
    table, free = s["table"].cpu().numpy().copy(), s["free"].cpu().numpy()
    lens, new = s["lens"].tolist(), s["new"].tolist()
    head = first = s["head"].tolist()[0]
    positions, slots = [0] * s["tokens"], [-1] * s["tokens"]
    granted, offsets, short = [], [0], False
    for b, (have, n) in enumerate(zip(lens, new)):
        at = offsets[-1]
        offsets.append(at + n)
        lo, hi = -(-have // PAGE), -(-(have + n) // PAGE)
        good = hi <= table.shape[1] and at + n <= s["tokens"]
        if good and hi > lo:
            short = short or head + hi - lo > len(free)
            good = not short
        if good:
            table[b, lo:hi] = free[head: head + hi - lo]
            head += hi - lo
        granted.append(n if good else 0)
        for j in range(min(n, s["tokens"] - at)):
            p = have + j
            positions[at + j] = p
            if good:
                slots[at + j] = int(table[b, p // PAGE]) * PAGE + p % PAGE
    assert head >= first
    dev = s["table"].device
    return [torch.from_numpy(table).to(dev), _i32([a + g for a, g in zip(lens, granted)]), _i32([head]), _i32(offsets),
            _i32(positions), torch.tensor(slots, device=dev), _i32(granted)]


def _exact_rope(s: dict):
    c = s["case"]
    d, rot = c["dim"], c["rot"]
    # one complex number per pair, turned by e^(i pos f)
    if c["layout"] == "interleaved":
        re, im = torch.arange(0, rot, 2, device=DEVICE), torch.arange(1, rot, 2, device=DEVICE)
    else:
        re, im = torch.arange(0, rot // 2, device=DEVICE), torch.arange(rot // 2, rot, device=DEVICE)
    angle = s["pos"].to(torch.float64).outer(s["freq"])
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle).unsqueeze(1)

    def rotate(x):
        y = x.to(torch.float64).contiguous()
        z = torch.complex(y[..., re], y[..., im]) * turn
        y[..., re], y[..., im] = z.real, z.imag
        return y

    flat = lambda pool: pool.to(torch.float64).transpose(1, 2).reshape(-1, c["kv_heads"], d)
    back = lambda rows: rows.reshape(-1, PAGE, c["kv_heads"], d).transpose(1, 2).contiguous()
    kp, vp = flat(s["k_pool"]), flat(s["v_pool"])
    kp[s["slots"]] = rotate(s["k"])
    vp[s["slots"]] = s["v"].to(torch.float64)
    return [rotate(s["q"]), back(kp), back(vp)]


def _exact_shared(s: dict):
    hq, d = s["q"].shape[1:]
    hk = s["k_pool"].shape[1]
    rows = []
    for b, n in enumerate(s["host_lens"]):
        t = torch.arange(n, device=DEVICE)
        page = s["table"][b].long()[t // PAGE]
        heads = []
        for h in range(hk):
            k = s["k_pool"][page, h, t % PAGE].to(torch.float64)
            v = s["v_pool"][page, h, t % PAGE].to(torch.float64)
            q = s["q"][b, h * (hq // hk): (h + 1) * (hq // hk)].to(torch.float64)
            heads.append(torch.softmax((q @ k.T) * s["scale"], dim=-1) @ v)
        rows.append(torch.cat(heads))
    return torch.stack(rows)


def _exact_logprobs(s: dict):
    rows, top = s["logits"].shape[0], s["case"]["top"]
    lps, hs, ids, alts = [], [], [], []
    for r0 in range(0, rows, 64):
        x = s["logits"][r0: r0 + 64].to(torch.float64)
        lp = torch.log_softmax(x, dim=1)
        lps.append(lp.gather(1, s["ids"][r0: r0 + 64, None]).squeeze(1))
        hs.append(-(lp.exp() * lp).sum(dim=1))
        # the highest values first, equal ones by index
        order = np.argsort(-x.cpu().numpy(), axis=1, kind="stable")[:, :top] if rows <= 128 else None
        if order is not None:
            ids.append(torch.from_numpy(order.copy()).to(x.device))
            alts.append(lp.gather(1, ids[-1]))
        else:
            alts.append(torch.sort(lp, dim=1, descending=True).values[:, :top])
    return [torch.cat(lps), torch.cat(hs), torch.cat(ids) if ids else None, torch.cat(alts)]


# -------------------------------------------------------------------- work -----
def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "tables":
        held, new = _lengths(case)
        pages = sum(-(-(h + n) // PAGE) - (-(-h // PAGE)) for h, n in zip(held, new))
        return {"bytes": 20 * len(held) + 8 * pages + 12 * sum(new), "flops": 4 * sum(new)}
    size = 2 if case.get("dtype", "f16") == "f16" else 4
    if kind == "rope":
        t, hq, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        return {"bytes": t * (2 * (hq + 2 * hk) * d * size + 12), "flops": t * (hq + hk) * case["rot"] * 3}
    if kind == "shared":
        hq, hk, d = case["heads"], case["kv_heads"], 128
        groups, prefixes = _groups(case)
        batch = sum(groups)
        suffix = _spread(batch, case["lo"], case["hi"], 3)
        seen = sum(n * p for n, p in zip(groups, prefixes)) + sum(suffix)
        kept = sum(prefixes) + sum(suffix)
        return {"bytes": kept * hk * d * 4 + batch * hq * d * 4, "flops": 4 * d * hq * seen}
    rows, vocab = case["rows"], case["vocab"]
    return {"bytes": rows * (vocab * size + 16 + 12 * case["top"]), "flops": 4 * rows * vocab}
