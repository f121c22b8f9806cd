"""Operators of a step that verifies trees of drafted tokens: what a program calls for each, over the sizes it meets.

Kinds of case, in the order of a step:
* ``tree``: from each drafted token's parent, the masks of what every token may see of its tree, and rotary positions.
* ``norm``: norms of q and k for each head, their rotary positions, and the append of k and v to the pages.
* ``attend``: attention of the drafted tokens over their sequence's paged context and their own ancestors.
* ``logits``: penalties for repeated tokens (those on a drafted token's path among them), biases and grammar masks.
* ``accept``: the drafted tokens that the model's own choices confirm, and their K and V moved behind the context.

Sizes and the trees' shapes are fixed by the case alone; values come from the seed.
"""
from __future__ import annotations

import math
import random
import zlib

import numpy as np
import torch

own = False
DEVICE = "cuda"


# ------------------------------------------------------------------ cases ------
def listed() -> list[dict]:
    return [
        # one request with a small tree: the smallest step
        dict(name="tree b1 26 nodes", kind="tree", batch=1, lo=26, hi=26, far=2000, shape="bushy"),
        # a full server, ragged trees
        dict(name="tree b128 to 200 nodes", kind="tree", batch=128, lo=1, hi=200, far=16000, shape="mixed"),
        # one token of the float32 tiny model
        dict(name="norm tiny f32 1", kind="norm", tokens=1, heads=4, kv_heads=2, dim=64, rot=64, layout="interleaved",
             scaling="none", theta=10000.0, far=64, page=16, dtype="f32"),
        # a chunk of a long-context prompt: halves, frequencies scaled by bands, far positions
        dict(name="norm half 4093 far", kind="norm", tokens=4093, heads=32, kv_heads=8, dim=128, rot=128, layout="half",
             scaling="bands", theta=1000000.0, far=131072, page=16, dtype="f16"),
        # the tiny model verifies a few tokens
        dict(name="attend tiny f32 b1", kind="attend", batch=1, lo=7, hi=7, near=90, far=90, heads=4, kv_heads=2, dim=64,
             page=16, shape="bushy", dtype="f32"),
        # a few requests, latency counts
        dict(name="attend b4 26 nodes", kind="attend", batch=4, lo=26, hi=26, near=300, far=3000, heads=32, kv_heads=8,
             dim=128, page=16, shape="bushy", dtype="f16"),
        # a full server with small trees over ragged contexts
        dict(name="attend b32 to 16 nodes", kind="attend", batch=32, lo=5, hi=16, near=64, far=7168, heads=28, kv_heads=4,
             dim=128, page=16, shape="mixed", dtype="f16"),
        # large trees over long documents
        dict(name="attend b8 64 nodes long", kind="attend", batch=8, lo=57, hi=64, near=11000, far=16000, heads=32,
             kv_heads=8, dim=128, page=16, shape="bushy", dtype="f16"),
        # a decode step of 32 requests: answers of up to 8000 tokens, biases, one of three bound to a grammar
        dict(name="logits decode b32", kind="logits", batch=32, lo=1, hi=1, vocab=128256, near=40, far=8000, bias=64,
             allowed=True, shape="chain", dtype="f32"),
        # every node of large trees, logits in half precision
        dict(name="logits b8 trees of 64 f16", kind="logits", batch=8, lo=57, hi=64, vocab=152064, near=500, far=4000,
             bias=0, allowed=True, shape="bushy", dtype="f16"),
        # one request of the tiny model's size
        dict(name="accept b1 26 nodes", kind="accept", batch=1, lo=26, hi=26, near=90, far=90, layers=4, kv_heads=2,
             dim=64, page=16, depth=8, shape="bushy", dtype="f32"),
        # a full server: the K and V of all layers
        dict(name="accept b32 64 nodes", kind="accept", batch=32, lo=40, hi=64, near=3, far=100, layers=32, kv_heads=8,
             dim=128, page=16, depth=8, shape="bushy", dtype="f16"),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["tree", "norm", "norm", "attend", "attend", "attend", "logits", "logits", "accept", "accept"])
    shape = rng.choice(["bushy", "mixed", "chain"])
    if kind == "tree":
        hi = _log(rng, 1, 200)
        return dict(kind=kind, batch=_log(rng, 1, 128), lo=rng.randint(1, hi), hi=hi, far=_log(rng, 10, 16000),
                    shape=shape)
    if kind == "norm":
        heads, kv_heads, dim = rng.choice([(32, 8, 128), (28, 4, 128), (4, 2, 64), (16, 8, 96), (8, 8, 80), (8, 1, 256)])
        return dict(kind=kind, tokens=_log(rng, 1, 4096), heads=heads, kv_heads=kv_heads, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2, dim // 4]), layout=rng.choice(["interleaved", "half"]),
                    scaling=rng.choice(["none", "linear", "bands"]), theta=rng.choice([10000.0, 500000.0, 1000000.0]),
                    far=_log(rng, 64, 131072), page=rng.choice([16, 16, 32]), dtype=rng.choice(["f16", "f16", "f32"]))
    if kind == "attend":
        heads, kv_heads, dim, dtype = rng.choice([
            (32, 8, 128, "f16"), (28, 4, 128, "f16"), (16, 8, 128, "f16"), (8, 8, 128, "f16"), (16, 1, 128, "f16"),
            (4, 2, 64, "f32"), (16, 8, 96, "f32")])
        room = 220000000 // heads if dtype == "f16" else 4000000 // heads  # pairs of a drafted token and one it sees
        batch, hi = _log(rng, 1, 64), _log(rng, 1, 200)
        far = max(1, min(_log(rng, 20, 16000), room // batch // hi - hi, 1000000 // kv_heads // batch))
        return dict(kind=kind, batch=batch, lo=rng.randint(1, hi), hi=hi, near=rng.randint(0, far), far=far, heads=heads,
                    kv_heads=kv_heads, dim=dim, page=rng.choice([16, 16, 32]), shape=shape, dtype=dtype)
    if kind == "logits":
        vocab = rng.choice([1024, 16384, 128256, 152064, _log(rng, 100, 152064)])
        most = max(1, 70000000 // vocab)
        hi = rng.choice([1, min(_log(rng, 1, 200), most)])
        far = _log(rng, 1, 16000)
        return dict(kind=kind, batch=_log(rng, 1, max(1, min(256, most // hi))), lo=rng.randint(1, hi), hi=hi, vocab=vocab,
                    near=rng.randint(0, far), far=far, bias=rng.choice([0, 1, 33, min(300, vocab // 2)]),
                    allowed=rng.choice([True, False]), shape=shape, dtype=rng.choice(["f32", "f32", "f16"]))
    kv_heads, dim, layers, dtype = rng.choice([(8, 128, 32, "f16"), (4, 128, 28, "f16"), (2, 64, 4, "f32"), (8, 96, 3, "f16")])
    hi, far = _log(rng, 1, 64), _log(rng, 3, 100)
    return dict(kind=kind, batch=_log(rng, 1, 32), lo=rng.randint(1, hi), hi=hi, near=rng.randint(0, far), far=far,
                layers=layers, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 16, 32]), depth=rng.randint(1, 12),
                shape=shape, dtype=dtype)


def _spread(n: int, lo: int, hi: int, salt: int) -> list[int]:
    """n whole numbers spread evenly between lo and hi in an order of their own (fixed by the case)."""
    v = [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(n * 1000003 + lo * 1009 + hi * 31 + salt).shuffle(v)
    return v


def _nodes(case: dict) -> list[int]:
    return _spread(case["batch"], case["lo"], case["hi"], 1)


def _words(case: dict) -> int:
    return -(-case["hi"] // 64)


def _parents(n: int, shape: str, salt: int) -> list[int]:
    """A tree of n drafted tokens in an order in which parents come first; the first one is the root.  "chain": one
    line of tokens; "bushy": a wide first level, few children further down; "mixed": some of each."""
    rng = random.Random(n * 7919 + salt)
    if shape == "mixed":
        shape = rng.choice(["chain", "bushy"])
    if shape == "chain":
        return [i - 1 for i in range(n)]
    first = max(1, n // 3)  # children of the root
    return [-1] + [0 if i <= first else rng.randint(max(1, i - first), i - 1) for i in range(1, n)]


# ------------------------------------------------------------------ values -----
def _gen(seed: int, *what) -> torch.Generator:
    g = torch.Generator(device=DEVICE)
    g.manual_seed((seed * 2654435761 + zlib.crc32(repr(what).encode())) & 0x7FFFFFFFFFFF)
    return g


def _randn(shape, seed: int, *what, dtype=torch.float32) -> torch.Tensor:
    return torch.randn(shape, generator=_gen(seed, *what), device=DEVICE, dtype=torch.float32).to(dtype)


def _rand(shape, seed: int, *what) -> torch.Tensor:
    return torch.rand(shape, generator=_gen(seed, *what), device=DEVICE)


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


def _contexts(case: dict) -> list[int]:
    return _spread(case["batch"], case["near"], case["far"], 2)


def _trees(case: dict) -> dict:
    """What a step keeps of its trees: parents, where each row's tokens begin, and their count."""
    nodes = _nodes(case)
    parents = [p for b, n in enumerate(nodes) for p in _parents(n, case["shape"], b)]
    return dict(nodes=nodes, parents=_i32(parents), offsets=_i32(np.cumsum([0] + nodes).tolist()), counts=_i32(nodes))


def _table(lens: list[int], page: int, seed: int) -> tuple[torch.Tensor, int]:
    """Page tables of sequences of these lengths, pages in any order, and the number of pages."""
    pages = [-(-n // page) for n in lens]
    width, used = max(pages), sum(pages)
    first = np.cumsum([0] + pages)
    at = np.minimum(first[:-1, None] + np.arange(width)[None, :], first[1:, None] - 1)
    order = torch.randperm(used, generator=_gen(seed, "pages"), device=DEVICE).to(torch.int32)
    return order[torch.from_numpy(at).to(DEVICE)].contiguous(), used


def _host_masks(nodes: list[int], shape: str, words: int) -> torch.Tensor:
    """Bit k of row j: token k of the same tree is j or one of its ancestors."""
    rows = []
    for b, n in enumerate(nodes):
        seen: list[int] = []
        for i, p in enumerate(_parents(n, shape, b)):
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        rows += [[(m >> 64 * w) & 0xFFFFFFFFFFFFFFFF for w in range(words)] for m in seen]
    return torch.from_numpy(np.array(rows, dtype=np.uint64).reshape(-1, words).view(np.int64)).to(DEVICE)


def prepare(case: dict, seed: int) -> dict:
    return dict(tree=_prepare_tree, norm=_prepare_norm, attend=_prepare_attend, logits=_prepare_logits,
                accept=_prepare_accept)[case["kind"]](case, seed)


def _prepare_tree(case: dict, seed: int) -> dict:
    t = _trees(case)
    ctx = torch.randint(0, case["far"] + 1, (case["batch"],), generator=_gen(seed, "ctx"), device=DEVICE)
    return dict(case=case, lens=(ctx + t["counts"]).to(torch.int32), words=_words(case), most=case["hi"], **t)


def _prepare_norm(case: dict, seed: int) -> dict:
    t, hq, hk, d, p = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "page"))
    dt = _dtype(case)
    q, k, v = (1.5 * _randn((t, (hq + 2 * hk) * d), seed, "qkv")).to(dt).split([hq * d, hk * d, hk * d], dim=1)
    pages = -(-t // p) + 3
    freq, factor = _frequencies(case)
    return dict(case=case, q=q.unflatten(1, (hq, d)), k=k.unflatten(1, (hk, d)), v=v.unflatten(1, (hk, d)),
                q_weight=(1.0 + 0.2 * _randn((d,), seed, "qw")).to(dt), k_weight=(1.0 + 0.2 * _randn((d,), seed, "kw")).to(dt),
                pos=torch.randint(0, case["far"], (t,), generator=_gen(seed, "pos"), device=DEVICE, dtype=torch.int32),
                slots=torch.randperm(pages * p, generator=_gen(seed, "slots"), device=DEVICE)[:t],
                freq=torch.tensor(freq, dtype=torch.float64, device=DEVICE), factor=factor, eps=1e-6,
                k_pool=torch.zeros((pages, hk, p, d), dtype=dt, device=DEVICE),
                v_pool=torch.zeros((pages, hk, p, d), dtype=dt, device=DEVICE))


def _prepare_attend(case: dict, seed: int) -> dict:
    hq, hk, d, p, dt = case["heads"], case["kv_heads"], case["dim"], case["page"], _dtype(case)
    t = _trees(case)
    lens = [c + n for c, n in zip(_contexts(case), t["nodes"])]
    table, used = _table(lens, p, seed)
    return dict(case=case, q=_randn((sum(t["nodes"]), hq, d), seed, "q", dtype=dt),
                k_pool=_randn((used, hk, p, d), seed, "k", dtype=dt), v_pool=_randn((used, hk, p, d), seed, "v", dtype=dt),
                table=table, lens=_i32(lens), longest=max(lens), most=case["hi"], scale=1.0 / math.sqrt(d),
                masks=_host_masks(t["nodes"], case["shape"], _words(case)), **t)


def _prepare_logits(case: dict, seed: int) -> dict:
    b, vocab = case["batch"], case["vocab"]
    t = _trees(case)
    rows = sum(t["nodes"])
    # logits of a model: a wide bulk and a few likely tokens
    x = _randn((rows, vocab), seed, "logits") * 2.5
    likely = torch.randint(0, vocab, (rows, 12), generator=_gen(seed, "likely"), device=DEVICE)
    x.scatter_add_(1, likely, 9.0 + 2.0 * _randn((rows, 12), seed, "peaks"))
    x = x.to(_dtype(case))
    held = _contexts(case)
    words = lambda what, *shape: (vocab * _rand(shape, seed, what) ** 3).long().clamp_(0, vocab - 1)  # some far more often
    state = dict(case=case, logits=x, out=torch.empty_like(x), history=words("history", b, max(1, case["far"])),
                 held=_i32(held), prompt=_i32([h // 3 for h in held]), drafts=words("drafts", rows), most=case["hi"],
                 masks=_host_masks(t["nodes"], case["shape"], _words(case)),
                 repetition=1.0 + 0.3 * _rand((b,), seed, "rep"), presence=0.5 * _rand((b,), seed, "pres"),
                 frequency=0.2 * _rand((b,), seed, "freq"), bias_ids=None, bias=None, allowed=None, **t)
    if case["bias"]:  # lists of their own lengths, the unused end marked by -1
        k = case["bias"]
        order = _rand((b, min(vocab, 4096)), seed, "bias ids").argsort(dim=1)[:, :k] * max(1, vocab // 4096)
        used = torch.randint(0, k + 1, (b, 1), generator=_gen(seed, "used"), device=DEVICE)
        state["bias_ids"] = torch.where(torch.arange(order.shape[1], device=DEVICE) < used, order, -1).contiguous()
        state["bias"] = 4.0 * _randn(tuple(order.shape), seed, "bias")
    if case["allowed"]:  # every third row free, the others with half or few of the tokens
        shape = (rows, -(-vocab // 32))
        bits = torch.randint(-2 ** 31, 2 ** 31, (4,) + shape, generator=_gen(seed, "allowed"), device=DEVICE, dtype=torch.int64)
        kind = torch.arange(rows, device=DEVICE)[:, None] % 3
        few = bits[0] & bits[1] & bits[2] & bits[3]
        state["allowed"] = torch.where(kind == 0, -1, torch.where(kind == 1, bits[0], few)).to(torch.int32)
    return state


def _prepare_accept(case: dict, seed: int) -> dict:
    hk, d, p, dt, vocab, depth = case["kv_heads"], case["dim"], case["page"], _dtype(case), 32000, case["depth"]
    t = _trees(case)
    lens = [c + n for c, n in zip(_contexts(case), t["nodes"])]
    table, used = _table(lens, p, seed)
    rng = random.Random(seed * 31 + 7)
    drafts, targets = [], []
    for b, n in enumerate(t["nodes"]):
        parents = _parents(n, case["shape"], b)
        token = [rng.randrange(vocab) for _ in range(n)]
        target = [rng.randrange(vocab, 2 * vocab) for _ in range(n)]  # confirms none
        children = [[c for c in range(1, n) if parents[c] == i] for i in range(n)]
        path, stop = [0], rng.randint(1, depth + 2)
        while len(path) < stop:
            # (a step down to a token that a later pass over the same state finds where it was)
            kids = [c for c in children[path[-1]] if c == len(path) or c > depth + 2]
            if not kids:
                break
            path.append(rng.choice(kids))
            target[path[-2]] = token[path[-1]]
            for c in children[path[-2]]:  # siblings differ
                token[c] = token[c] if c == path[-1] else vocab * 3 + c
        drafts += token
        targets += target
    shape = (case["layers"], used, hk, p, d)
    long = lambda v: torch.tensor(v, dtype=torch.int64, device=DEVICE)
    return dict(case=case, lens=_i32(lens), table=table, drafts=long(drafts), targets=long(targets), most=case["hi"],
                k_pools=_randn(shape, seed, "k", dtype=dt), v_pools=_randn(shape, seed, "v", dtype=dt), **t)


# ------------------------------------------------------------------ passes -----
def run(state: dict):
    kind = state["case"]["kind"]
    return (_OWN if own else _PLAIN)[kind](state)


def _own_tree(s: dict):
    from cacheir_amd import kernels

    t = kernels.draft_tree(s["parents"], s["lens"], s["offsets"], s["counts"], words=s["words"])
    return [t.masks, t.positions]


def _own_norm(s: dict):
    from cacheir_amd import kernels

    q = kernels.norm_rope_append(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["eps"], s["pos"], s["slots"],
                                 s["freq"], s["k_pool"], s["v_pool"], layout=s["case"]["layout"], factor=s["factor"])
    return [q, s["k_pool"], s["v_pool"]]


def _own_attend(s: dict):
    from cacheir_amd import kernels

    return kernels.paged_tree_attention(s["q"], s["k_pool"], s["v_pool"], s["table"], s["lens"], s["offsets"],
                                        s["counts"], s["masks"], scale=s["scale"])


def _own_logits(s: dict):
    from cacheir_amd import kernels

    return kernels.adjust_logits(s["logits"], s["offsets"], history=s["history"], history_lens=s["held"],
                                 prompt_lens=s["prompt"], drafts=s["drafts"], masks=s["masks"],
                                 repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                                 bias_ids=s["bias_ids"], bias=s["bias"], allowed=s["allowed"], out=s["out"])


def _own_accept(s: dict):
    from cacheir_amd import kernels

    a = kernels.accept_drafts(s["parents"], s["drafts"], s["targets"], s["lens"], s["offsets"], s["counts"], s["table"],
                              s["k_pools"], s["v_pools"], most=s["case"]["depth"])
    return [a.accepted, a.path, a.tokens, a.seq_lens, s["k_pools"], s["v_pools"]]


def _padded(s: dict, tokens: torch.Tensor, fill: int) -> torch.Tensor:
    """Values of the drafted tokens as [row, token of its tree]."""
    col = torch.arange(s["most"], device=tokens.device)[None, :]
    at = torch.clamp(s["offsets"][:-1].long()[:, None] + col, max=tokens.shape[0] - 1)
    return torch.where(col < s["counts"][:, None], tokens[at].long(), fill)


def _rows_of(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """(row of each drafted token, its place in the row's tree)."""
    j = torch.arange(s["parents"].numel(), device=s["parents"].device)
    row = torch.searchsorted(s["offsets"].long(), j, right=True) - 1
    return row, j - s["offsets"].long()[row]


def _bits(masks: torch.Tensor, most: int) -> torch.Tensor:
    """[tokens, most] truth values of the masks' bits."""
    k = torch.arange(most, device=masks.device)
    return (masks[:, k // 64] >> (k % 64) & 1) != 0


def _plain_tree(s: dict):
    n, words = s["most"], s["words"]
    parents = _padded(s, s["parents"], -1)
    col = torch.arange(n, device=parents.device)
    above = ((parents[:, :, None] == col) | (col[:, None] == col)).float()  # [row, token, itself or its parent]
    for _ in range((n - 1).bit_length()):  # ancestors up to 1, 2, 4, ... steps away
        above = (torch.matmul(above, above) > 0).float()
    row, at = _rows_of(s)
    seen = above[row, at] > 0
    positions = (s["lens"] - s["counts"]).long()[row] + seen.sum(dim=1) - 1
    wide = torch.zeros((seen.shape[0], 64 * words), dtype=torch.int64, device=seen.device)
    wide[:, :n] = seen.long()
    masks = (wide.view(-1, words, 64) << torch.arange(64, device=seen.device)).sum(dim=2)
    return [masks, positions.int()]


def _plain_norm(s: dict):
    c = s["case"]
    rot, page = c["rot"], c["page"]
    turn = s["pos"].double()[:, None] * s["freq"][None, :]
    cos, sin = (torch.cos(turn) * s["factor"]).float()[:, None, :], (torch.sin(turn) * s["factor"]).float()[:, None, :]

    def turned(x, w):
        y = x.float()
        y = y * torch.rsqrt((y * y).mean(dim=2, keepdim=True) + s["eps"]) * w.float()
        if c["layout"] == "interleaved":
            a, b = y[..., 0:rot:2].clone(), y[..., 1:rot:2].clone()
            y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
        else:
            a, b = y[..., : rot // 2].clone(), y[..., rot // 2: rot].clone()
            y[..., : rot // 2], y[..., rot // 2: rot] = a * cos - b * sin, a * sin + b * cos
        return y.to(x.dtype)

    at, off = s["slots"] // page, s["slots"] % page
    s["k_pool"][at, :, off] = turned(s["k"], s["k_weight"])
    s["v_pool"][at, :, off] = s["v"]
    return [turned(s["q"], s["q_weight"]), s["k_pool"], s["v_pool"]]


def _plain_attend(s: dict):
    batch, hk, d, page = len(s["nodes"]), s["case"]["kv_heads"], s["case"]["dim"], s["case"]["page"]
    hq, n, longest = s["case"]["heads"], s["most"], s["longest"]
    g = hq // hk
    row, at = _rows_of(s)
    q = torch.zeros((batch, n, hq, d), device=s["q"].device)
    q[row, at] = s["q"].float()
    q = q.view(batch, n, hk, g, d).permute(0, 2, 1, 3, 4).reshape(batch, hk, n * g, d)
    pages = s["table"][:, : -(-longest // page)].long()
    rows = lambda pool: pool[pages].transpose(1, 2).reshape(batch, hk, -1, d)[:, :, :longest].float()
    token = torch.arange(longest, device=q.device)
    context = (s["lens"] - s["counts"]).long()[:, None]
    # token t of a row is part of the context, or drafted token t - context, which the masks' bits name
    bits = torch.zeros((batch, n, n), dtype=torch.bool, device=q.device)
    bits[row, at] = _bits(s["masks"], n)
    k = token[None, :] - context
    drafted = bits.gather(2, torch.clamp(k, 0, n - 1)[:, None, :].expand(batch, n, longest))
    seen = (k < 0)[:, None, :] | (drafted & (k < s["counts"][:, None])[:, None, :])
    w = torch.matmul(q, rows(s["k_pool"]).transpose(2, 3).contiguous()) * s["scale"]
    w = w.view(batch, hk, n, g, longest).masked_fill_(~seen[:, None, :, None, :], -math.inf).view(batch, hk, n * g, longest)
    w = torch.exp(w - w.amax(dim=3, keepdim=True).clamp(min=-1e30))
    o = torch.matmul(w, rows(s["v_pool"])) / w.sum(dim=3, keepdim=True)
    o = o.view(batch, hk, n, g, d).transpose(1, 2).reshape(batch, n, hq, d)
    return o[row, at].to(s["q"].dtype)


def _plain_logits(s: dict):
    rows, vocab = s["logits"].shape
    batch, dev = s["held"].numel(), s["logits"].device
    row, _ = _rows_of(s)
    col = torch.arange(s["history"].shape[1], device=dev)[None, :]
    held = (col < s["held"][:, None]).int()
    given = (col >= s["prompt"][:, None]).int() * held  # behind the prompt
    seen = torch.zeros((batch, vocab), dtype=torch.int32, device=dev).scatter_add_(1, s["history"], held)
    count = torch.zeros((batch, vocab), dtype=torch.int32, device=dev).scatter_add_(1, s["history"], given)
    path = _bits(s["masks"], s["most"]).int()  # the drafted tokens up to and with the row's own
    tokens = _padded(s, s["drafts"], 0)[row]
    count = count[row].scatter_add_(1, tokens, path)
    seen = seen[row] + count
    x = s["logits"].float()
    rep = s["repetition"][row][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][row][:, None] * count - s["presence"][row][:, None] * (count > 0)
    if s["bias"] is not None:
        extra = torch.zeros((batch, vocab + 1), device=dev)
        extra.scatter_(1, torch.where(s["bias_ids"] < 0, vocab, s["bias_ids"]), s["bias"])
        x = x + extra[row, :vocab]
    if s["allowed"] is not None:
        v = torch.arange(vocab, device=dev)
        x = torch.where((s["allowed"][:, v // 32] >> (v % 32).int() & 1) != 0, x, -math.inf)
    return x.to(s["logits"].dtype)


def _plain_accept(s: dict):
    depth, page = s["case"]["depth"], s["case"]["page"]
    parents, drafts, targets = _padded(s, s["parents"], -1), _padded(s, s["drafts"], -1), _padded(s, s["targets"], -2)
    batch, n = parents.shape
    col = torch.arange(n, device=parents.device)
    # fits[row, token, child]: the child is the model's choice after the token; the first one follows
    fits = (parents[:, None, :] == col[None, :, None]) & (drafts[:, None, :] == targets[:, :, None])
    follows = torch.where(fits, col, n).amin(dim=2)
    follows = torch.cat([follows, torch.full_like(follows[:, :1], n)], dim=1)
    path = torch.full((batch, depth), n, dtype=torch.int64, device=parents.device)
    path[:, 0] = 0
    for i in range(1, depth):
        path[:, i] = follows.gather(1, path[:, i - 1: i]).squeeze(1)
    taken = path < n
    accepted = taken.sum(dim=1)
    tokens = torch.where(taken, targets.gather(1, torch.clamp(path, max=n - 1)), -1)
    context = (s["lens"] - s["counts"]).long()[:, None]
    to = context + torch.where(taken, torch.arange(depth, device=path.device), 0)
    of = context + torch.where(taken, path, 0)
    slot = lambda at: (s["table"].gather(1, at // page).long(), at % page)
    (p0, o0), (p1, o1) = slot(of), slot(to)
    s["k_pools"][:, p1, :, o1] = s["k_pools"][:, p0, :, o0]
    s["v_pools"][:, p1, :, o1] = s["v_pools"][:, p0, :, o0]
    return [accepted.int(), torch.where(taken, path, -1).int(), tokens, (context.squeeze(1) + accepted).int(), s["k_pools"],
            s["v_pools"]]


_OWN = dict(tree=_own_tree, norm=_own_norm, attend=_own_attend, logits=_own_logits, accept=_own_accept)
_PLAIN = dict(tree=_plain_tree, norm=_plain_norm, attend=_plain_attend, logits=_plain_logits, accept=_plain_accept)


# -------------------------------------------------------------- references -----
def exact(case: dict, seed: int):
    """What ``run`` returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    return dict(tree=_exact_tree, norm=_exact_norm, attend=_exact_attend, logits=_exact_logits,
                accept=_exact_accept)[case["kind"]](s)


def _exact_tree(s: dict):
    shape, lens, positions = s["case"]["shape"], s["lens"].tolist(), []
    for b, n in enumerate(s["nodes"]):
        depth: list[int] = []
        for p in _parents(n, shape, b):
            depth.append(depth[p] + 1 if p >= 0 else 0)
        positions += [lens[b] - n + x for x in depth]
    return [_host_masks(s["nodes"], shape, s["words"]), _i32(positions)]


def _exact_norm(s: dict):
    c = s["case"]
    d, rot, page = c["dim"], c["rot"], c["page"]
    # one complex number per pair, turned by e^(i pos f)
    if c["layout"] == "interleaved":
        re, im = torch.arange(0, rot, 2, device=DEVICE), torch.arange(1, rot, 2, device=DEVICE)
    else:
        re, im = torch.arange(0, rot // 2, device=DEVICE), torch.arange(rot // 2, rot, device=DEVICE)
    angle = s["pos"].to(torch.float64).outer(s["freq"])
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle).unsqueeze(1)

    def turned(x, w):
        y = x.to(torch.float64).contiguous()
        y = y / (y.square().mean(dim=-1) + s["eps"]).sqrt().unsqueeze(-1) * w.to(torch.float64)
        z = torch.complex(y[..., re], y[..., im]) * turn
        y[..., re], y[..., im] = z.real, z.imag
        return y

    flat = lambda pool: pool.to(torch.float64).transpose(1, 2).reshape(-1, c["kv_heads"], d)
    back = lambda rows: rows.reshape(-1, page, c["kv_heads"], d).transpose(1, 2).contiguous()
    kp, vp = flat(s["k_pool"]), flat(s["v_pool"])
    kp[s["slots"]] = turned(s["k"], s["k_weight"])
    vp[s["slots"]] = s["v"].to(torch.float64)
    return [turned(s["q"], s["q_weight"]), back(kp), back(vp)]


def _exact_attend(s: dict):
    c = s["case"]
    hq, hk, page, first, lens, rows = c["heads"], c["kv_heads"], c["page"], 0, s["lens"].tolist(), []
    for b, n in enumerate(s["nodes"]):
        seen = torch.zeros((n, lens[b]), dtype=torch.bool)
        seen[:, : lens[b] - n] = True
        for i, p in enumerate(_parents(n, c["shape"], b)):
            if p >= 0:
                seen[i] = seen[p]
            seen[i, lens[b] - n + i] = True
        seen = seen.to(DEVICE)[None].expand(hq // hk, n, lens[b])
        t = torch.arange(lens[b], device=DEVICE)
        at = s["table"][b].long()[t // page]
        heads = []
        for h in range(hk):
            k = s["k_pool"][at, h, t % page].to(torch.float64)
            v = s["v_pool"][at, h, t % page].to(torch.float64)
            q = s["q"][first: first + n, h * (hq // hk): (h + 1) * (hq // hk)].to(torch.float64).transpose(0, 1)
            x = ((q.reshape(-1, q.shape[2]) @ k.T) * s["scale"]).reshape(seen.shape)
            w = torch.softmax(torch.where(seen, x, -math.inf), dim=-1)
            heads.append((w.reshape(-1, lens[b]) @ v).reshape(q.shape))
        rows.append(torch.cat(heads).transpose(0, 1))
        first += n
    return torch.cat(rows)


def _exact_logits(s: dict):
    vocab, first, out = s["case"]["vocab"], 0, []
    for b, n in enumerate(s["nodes"]):
        held, prompt = int(s["held"][b]), int(s["prompt"][b])
        all_of = torch.bincount(s["history"][b, :held], minlength=vocab)
        mine = torch.bincount(s["history"][b, prompt:held], minlength=vocab)
        bias = torch.zeros(vocab, dtype=torch.float64, device=DEVICE)
        if s["bias"] is not None:
            use = s["bias_ids"][b] >= 0
            bias[s["bias_ids"][b][use]] = s["bias"][b][use].to(torch.float64)
        rep, freq, pres = (float(s[k][b]) for k in ("repetition", "frequency", "presence"))
        parents = _parents(n, s["case"]["shape"], b)
        for i in range(n):
            path, k = [], i
            while k >= 0:
                path.append(k)
                k = parents[k]
            extra = torch.bincount(s["drafts"][first: first + n][path], minlength=vocab)
            x = s["logits"][first + i].to(torch.float64)
            x = torch.where(all_of + extra > 0, torch.where(x > 0, x / rep, x * rep), x)
            x = x - freq * (mine + extra) - pres * (mine + extra).clamp(max=1) + bias
            if s["allowed"] is not None:
                bits = s["allowed"][first + i][:, None] >> torch.arange(32, device=DEVICE, dtype=torch.int32)[None, :]
                x = x.masked_fill((bits & 1).reshape(-1)[:vocab] == 0, -math.inf)
            out.append(x)
        first += n
    return torch.stack(out)


def _exact_accept(s: dict):
    c, first = s["case"], 0
    table, drafts, targets, lens = s["table"].tolist(), s["drafts"].tolist(), s["targets"].tolist(), s["lens"].tolist()
    accepted, paths, tokens, ends, of, to = [], [], [], [], [], []
    for b, n in enumerate(s["nodes"]):
        parents = _parents(n, c["shape"], b)
        path = [0]
        while len(path) < c["depth"]:
            kids = [k for k in range(n) if parents[k] == path[-1] and drafts[first + k] == targets[first + path[-1]]]
            if not kids:
                break
            path.append(kids[0])
        start = lens[b] - n
        for i, k in enumerate(path):
            of.append((table[b][(start + k) // c["page"]], (start + k) % c["page"]))
            to.append((table[b][(start + i) // c["page"]], (start + i) % c["page"]))
        pad = [-1] * (c["depth"] - len(path))
        accepted.append(len(path))
        paths.append(path + pad)
        tokens.append([targets[first + k] for k in path] + pad)
        ends.append(start + len(path))
        first += n
    (p0, o0), (p1, o1) = (torch.tensor(x, device=DEVICE).T for x in (of, to))

    def moved(pools):
        flat = pools.clone().transpose(2, 3)  # [layer, page, offset, head, dim]
        flat[:, p1, o1] = pools.transpose(2, 3)[:, p0, o0]
        return flat.transpose(2, 3)

    return [_i32(accepted), _i32(paths), torch.tensor(tokens, device=DEVICE), _i32(ends), moved(s["k_pools"]),
            moved(s["v_pools"])]


# -------------------------------------------------------------------- work -----
def work(case: dict) -> dict:
    kind = case["kind"]
    size = 2 if case.get("dtype", "f16") == "f16" else 4
    if kind == "norm":
        t, hq, hk, d = (case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
        return {"bytes": t * (2 * (hq + 2 * hk) * d * size + 12), "flops": t * (hq + hk) * (4 * d + 3 * case["rot"])}
    nodes = _nodes(case)
    if kind == "tree":
        return {"bytes": 8 * len(nodes) + sum(nodes) * (8 + 8 * _words(case)), "flops": sum(nodes)}
    held = _contexts(case)
    if kind == "attend":
        hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
        return {"bytes": sum(c + n for c, n in zip(held, nodes)) * hk * d * 2 * size + sum(nodes) * hq * d * 2 * size,
                "flops": 4 * d * hq * sum(n * (c + n) for c, n in zip(held, nodes))}
    if kind == "logits":
        rows, vocab = sum(nodes), case["vocab"]
        return {"bytes": rows * vocab * 2 * size + 8 * sum(held) + 12 * case["bias"] * len(nodes) +
                (rows * vocab // 8 if case["allowed"] else 0), "flops": 6 * rows * vocab}
    # the path is not known before: at most `depth` tokens a row move, in every layer
    moved = sum(min(n, case["depth"]) - 1 for n in nodes)
    return {"bytes": moved * case["layers"] * case["kv_heads"] * case["dim"] * 4 * size + 20 * sum(nodes),
            "flops": sum(nodes)}
