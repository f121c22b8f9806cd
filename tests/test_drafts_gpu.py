"""The operators of a step that verifies trees of drafted tokens, against plain 64-bit implementations on the CPU: tree
masks, norm + rotary append, tree attention, logit penalties and masks, acceptance, and a run of them together.

Tolerances are sums of the roundings that the kernels make (u16 = 2^-11 and u32 = 2^-24: half a step of fp16 and fp32,
relative to the value):
* attention in fp16: each weight is rounded to fp16 once and the sum takes the rounded ones (2 u16 of sum w |v|, or 2^-25 / l
  per token for weights below fp16's normal range), scores are fp32 sums of at most 256 products (an exponent off by 260 u32
  |scale| sum |q k|, twice), the output is rounded to fp16 once more (u16 |out|); in fp32: the exponents, (n + 64) u32 of
  sum w |v| for the sums over n tokens, their joins and the exponentials, 2 u32 |out|;
* norm + rotary: a sum of squares of d terms and its root (d / 2 + 8 u32, relative), two products (2 u32), the reduced angle
  (pi u32) and sine and cosine (4 u32): (d / 2 + 22) u32 factor (|a| + |b|) in all with the products of the turn, plus the
  rounding to the output type;
* logits: a quotient or product, an FMA, two sums: 4 u32 of the magnitudes summed, plus the rounding to the output type.
Masks, positions, paths, tokens, lengths, pages and moved values are exact.
"""
import math
import random

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U16, U32 = 2.0 ** -11, 2.0 ** -24


def i32(v):
    return torch.tensor(v, dtype=torch.int32)


def tree(n, seed, shape="any"):
    rng = random.Random(seed)
    if shape == "chain":
        return [i - 1 for i in range(n)]
    if shape == "flat":
        return [-1 if i == 0 else 0 for i in range(n)]
    if shape == "forest":  # several tokens follow the context
        return [rng.randint(-1, i - 1) for i in range(n)]
    return [rng.randint(max(0, i - 9), i - 1) if i else -1 for i in range(n)]


def seen_sets(parents):
    """Python integers: bit k set where k is the token or an ancestor."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if 0 <= p < i else 0) | 1 << i)
    return out


def mask_words(sets, words):
    rows = [[(m >> 64 * w) & (2 ** 64 - 1) for w in range(words)] for m in sets]
    return torch.from_numpy(np.array(rows, dtype=np.uint64).reshape(-1, words).view(np.int64).copy())


# ------------------------------------------------------------------- masks -----
@pytest.mark.parametrize("words", [1, 2, 3, 4])
@pytest.mark.parametrize("shape", ["chain", "flat", "forest", "any"])
def test_draft_tree(device, words, shape):
    from cacheir_amd import kernels

    top = 64 * words
    nodes = [1, top, 0, 2, top - 1, 33, 63, 64, top // 2 + 1]
    gaps = [0, 0, 3, 0, 1, 0, 0, 2, 5]  # tokens of rows that were not granted, or not all
    parents, masks, positions, offsets, counts, lens = [], [], [], [0], [], []
    for b, (n, gap) in enumerate(zip(nodes, gaps)):
        n = min(n, top)
        p = tree(n, b, shape)
        sets = seen_sets(p)
        lens.append(n + [0, 5, 1000, 131072][b % 4])
        parents += p + [0] * gap
        masks += sets + [0] * gap
        positions += [lens[-1] - n + bin(m).count("1") - 1 for m in sets] + [0] * gap
        counts.append(n)
        offsets.append(len(parents))
    parents += [-1] * 7  # past the last row
    masks += [0] * 7
    positions += [0] * 7
    got = kernels.draft_tree(*(i32(x).to(device) for x in (parents, lens, offsets, counts)), words=words)
    assert torch.equal(got.masks.cpu(), mask_words(masks, words))
    assert got.positions.tolist() == positions


def test_draft_tree_of_odd_numbers(device):
    """Parents that do not lie before their token stand for none; counts and offsets past the tokens are cut."""
    from cacheir_amd import kernels

    dev = lambda *v: [i32(x).to(device) for x in v]
    t = kernels.draft_tree(*dev([5, 1, 2, -7, 2, 0], [6], [0, 6], [6]), words=1)
    assert t.masks.squeeze(1).tolist() == [1, 2, 4, 8, 4 | 16, 1 | 32] and t.positions.tolist() == [0, 0, 0, 0, 1, 1]
    t = kernels.draft_tree(*dev([-1, 0, 1], [9, 9], [0, 2, 9], [5, 7]), words=1)
    assert t.masks.squeeze(1).tolist() == [1, 3, 1] and t.positions.tolist() == [7, 8, 8]
    t = kernels.draft_tree(*dev([-1, 0, 1], [9, 9], [-4, -2, -1], [2, 1]), words=1)
    assert t.masks.abs().sum() == 0 and t.positions.tolist() == [0, 0, 0]
    t = kernels.draft_tree(*dev(list(range(-1, 99)), [100], [0, 100], [100]), words=1)  # past the masks' 64
    assert t.positions.tolist()[:64] == list(range(36, 100)) and t.positions.tolist()[64:] == [0] * 36
    t = kernels.draft_tree(*dev([], [4], [0, 0], [0]), words=1)
    assert t.masks.shape == (0, 1)


@pytest.mark.parametrize("words", [1, 2, 4])
def test_draft_tree_rows_past_their_masks(device, words):
    """A row of more tokens than its masks have bits for is refused: all of its masks are empty; other rows are as ever."""
    from cacheir_amd import kernels

    top = 64 * words
    nodes, parents, masks, offsets = [3, top + 1, top, 2 * top + 9, 5], [], [], [0]
    for b, n in enumerate(nodes):
        p = tree(n, b)
        parents += p
        masks += seen_sets(p) if n <= top else [0] * n
        offsets.append(len(parents))
    lens = [n + 40 for n in nodes]
    got = kernels.draft_tree(*(i32(x).to(device) for x in (parents, lens, offsets, nodes)), words=words)
    assert torch.equal(got.masks.cpu(), mask_words(masks, words))
    live = [j for b, n in enumerate(nodes) if n <= top for j in range(offsets[b], offsets[b + 1])]
    assert [got.positions.tolist()[j] for j in live] == [39 + bin(masks[j]).count("1") for j in live]


# --------------------------------------------------------------- attention -----
def tree_case(seed, nodes, contexts, hq, hkv, d=128, psize=16, words=1, dtype=torch.float16, shape="any", gaps=None,
              extra=2):
    """CPU tensors of a call; ``gaps``: query rows that no row counts, behind each row's."""
    g = torch.Generator().manual_seed(seed)
    lens = [c + n for c, n in zip(contexts, nodes)]
    pages = [-(-x // psize) for x in lens]
    width = max(max(pages), 1) + 1
    perm = torch.randperm(sum(pages) + extra, generator=g)
    table, at = torch.zeros((len(nodes), width), dtype=torch.int32), 0
    for b, p in enumerate(pages):
        table[b, :p] = perm[at: at + p].int()
        at += p
    gaps = gaps or [0] * len(nodes)
    sets, offsets = [], [0]
    for b, (n, gap) in enumerate(zip(nodes, gaps)):
        sets += seen_sets(tree(n, seed * 100 + b, shape)) + [0] * gap
        offsets.append(len(sets))
    randn = lambda *s: torch.randn(s, generator=g).to(dtype)
    used = sum(pages) + extra
    return dict(q=randn(len(sets), hq, d), k_pool=randn(used, hkv, psize, d), v_pool=randn(used, hkv, psize, d),
                page_table=table, seq_lens=i32(lens), offsets=i32(offsets), counts=i32(nodes), masks=mask_words(sets, words))


def bits_of(masks, n):
    k = torch.arange(n)
    return (masks[:, k // 64] >> (k % 64) & 1) != 0


def attention64(c, scale):
    """(out, tolerance) in float64; rows that no sequence counts are NaN."""
    q, kp, vp = c["q"].double(), c["k_pool"].double(), c["v_pool"].double()
    hq, d = q.shape[1:]
    hkv, psize = kp.shape[1], kp.shape[2]
    out, tol = torch.full_like(q, math.nan), torch.zeros_like(q)
    for b, n in enumerate(c["counts"].tolist()):
        first, length = int(c["offsets"][b]), int(c["seq_lens"][b])
        if n == 0:
            continue
        t = torch.arange(length)
        pages = c["page_table"][b].long()[t // psize]
        seen = torch.cat([torch.ones((n, length - n), dtype=torch.bool), bits_of(c["masks"][first: first + n], n)], dim=1)
        for i in range(n):
            at = t[seen[i]]
            if at.numel() == 0:
                out[first + i] = 0.0
                continue
            for h in range(hkv):
                g = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                k, v = kp[pages[at], h, at % psize], vp[pages[at], h, at % psize]
                s = q[first + i, g] @ k.T * scale
                e = torch.exp(s - s.max(dim=1, keepdim=True).values)
                l = e.sum(dim=1, keepdim=True)
                w = e / l
                o = w @ v
                off = 260 * U32 * abs(scale) * (q[first + i, g].abs() @ k.abs().T).max(dim=1, keepdim=True).values
                mass = w @ v.abs()
                out[first + i, g] = o
                if c["q"].dtype == torch.float16:
                    tol[first + i, g] = mass * (2 * U16 + 2 * off) + v.abs().sum(dim=0) * 2.0 ** -25 / l + U16 * o.abs()
                else:
                    tol[first + i, g] = mass * (2 * off + (at.numel() + 64) * U32) + 2 * U32 * o.abs()
    return out, tol


def run_tree(c, device, scale=None, **kw):
    from cacheir_amd import kernels

    return kernels.paged_tree_attention(**{k: v.to(device) for k, v in c.items()}, scale=scale, **kw)


def check_tree(c, got, scale=None):
    scale = c["q"].shape[2] ** -0.5 if scale is None else scale
    ref, tol = attention64(c, scale)
    live = ~ref.isnan()
    err = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got.cpu()[live]).all()
    assert bool((err[live] <= tol[live]).all()), f"max excess {(err - tol)[live].max():.3e}, error {err[live].max():.3e}"


@pytest.mark.parametrize("hq,hkv,nodes,contexts,psize", [
    (8, 2, [1], [0], 16),                                    # one token that sees itself
    (8, 2, [1], [1], 16),
    (32, 8, [26, 7, 1, 64], [500, 33, 1000, 4], 16),         # 104, 28, 4 and 256 vectors
    (28, 4, [16] * 5, [0, 31, 32, 33, 700], 16),             # 112 vectors, drafted tokens across blocks
    (32, 8, [8, 16, 32, 9, 17], [95, 300, 17, 1023, 64], 32),  # whole tiles of 32, 64 and 128, and a little more
    (16, 1, [3, 20, 64], [640, 1, 77], 48),
    (32, 1, [2, 33], [40, 100], 64),                         # 32 query heads on one KV head
    (8, 8, [40, 1, 12, 64], [64, 333, 0, 2000], 16),
    (4, 4, [3, 31, 32], [1, 2, 3], 128),
    (64, 1, [5, 40], [100, 9], 16),                          # 64 query heads on one KV head
    (5, 1, [13, 50], [200, 61], 16),
])
def test_tree_attention_shapes(device, hq, hkv, nodes, contexts, psize):
    c = tree_case(hq + len(nodes), nodes, contexts, hq, hkv, psize=psize)
    check_tree(c, run_tree(c, device, check_tables=True))


@pytest.mark.parametrize("seed", range(10))
def test_tree_attention_random(device, seed):
    rng = np.random.default_rng(seed)
    hq, hkv = [(32, 8), (28, 4), (16, 8), (6, 2), (12, 1)][seed % 5]
    rows, words = int(rng.integers(1, 7)), int(rng.integers(1, 5))
    nodes = [int(x) for x in rng.integers(0, int(rng.choice([3, 20, 64 * words])) + 1, rows)]
    contexts = [int(x) for x in rng.integers(0, int(rng.choice([3, 100, 900])), rows)]
    gaps = [int(x) for x in rng.integers(0, 3, rows)]
    if sum(nodes) + sum(gaps) == 0:
        gaps[0] = 2
    c = tree_case(seed, nodes, contexts, hq, hkv, psize=int(rng.choice([16, 32])), words=words, gaps=gaps,
                  shape=["any", "chain", "forest", "flat"][seed % 4])
    check_tree(c, run_tree(c, device))


@pytest.mark.parametrize("hq,hkv,d,psize,dtype", [
    (4, 2, 64, 16, torch.float32), (4, 4, 1, 16, torch.float32), (6, 2, 40, 7, torch.float32), (8, 1, 80, 16, torch.float16),
    (3, 3, 96, 5, torch.float32), (16, 2, 256, 16, torch.float16), (4, 1, 255, 16, torch.float32),
    (8, 2, 128, 16, torch.float32), (8, 2, 128, 8, torch.float16), (2, 2, 129, 1, torch.float32), (8, 2, 64, 16, torch.float16)])
def test_tree_attention_other_sizes(device, hq, hkv, d, psize, dtype):
    c = tree_case(d, [9, 1, 70, 0, 17], [150, 0, 3, 9, 600], hq, hkv, d=d, psize=psize, words=2, dtype=dtype,
                  gaps=[1, 0, 0, 2, 0])
    check_tree(c, run_tree(c, device, check_tables=True))
    check_tree(c, run_tree(c, device, scale=-0.3), scale=-0.3)


KINDS = [(32, 8, 128, torch.float16), (4, 2, 64, torch.float32), (8, 2, 64, torch.float16)]


@pytest.mark.parametrize("hq,hkv,d,dtype", KINDS)
def test_tree_attention_any_masks(device, hq, hkv, d, dtype):
    """Masks that are no trees: tokens that see others after them, not themselves, or nothing; bits past the row's
    tokens count for nothing."""
    nodes, contexts = [40, 64, 3, 5, 130], [70, 0, 0, 0, 0]
    c = tree_case(5, nodes, contexts, hq, hkv, d=d, words=3, dtype=dtype)
    g = torch.Generator().manual_seed(9)
    c["masks"] = torch.randint(-2 ** 62, 2 ** 62, c["masks"].shape, generator=g) * 2 + torch.randint(0, 2, c["masks"].shape, generator=g)
    c["masks"][50:60] = 0
    first = int(c["offsets"][2])
    c["masks"][first] = torch.tensor([-8, -1, -1])      # only bits past the row's three tokens
    c["masks"][first + 1] = torch.tensor([0, 0, 0])
    got = run_tree(c, device)
    check_tree(c, got)
    assert (got[first: first + 2] == 0).all() and (got[50:60] == 0).all()


@pytest.mark.parametrize("hq,hkv,d,dtype", KINDS)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_tree_attention_what_is_not_seen_does_not_count(device, hq, hkv, d, dtype, bad):
    """NaN and infinities in K and V of drafted tokens that a token does not see, behind the context and in unused pages;
    the tokens that do see them have them."""
    nodes, contexts = [30, 20, 1], [100, 7, 33]
    c = tree_case(3, nodes, contexts, hq, hkv, d=d, dtype=dtype)
    ref = run_tree(c, device).cpu()
    psize, tables, dirty = 16, c["page_table"], []
    for b, n in enumerate(nodes):
        first = int(c["offsets"][b])
        victims = [k for k in (n - 1, n - 4, n // 2) if k > 0]
        for which, k in enumerate(victims):
            pos = contexts[b] + k
            page, off = int(tables[b, pos // psize]), pos % psize
            if which != 1:
                c["k_pool"][page, :, off, :: 3] = bad
            if which != 2:
                c["v_pool"][page, :, off, 1:: 2] = bad
        hit = bits_of(c["masks"][first: first + n], n)[:, victims].any(dim=1) if victims else torch.zeros(n, dtype=torch.bool)
        dirty.append(hit)
        last = contexts[b] + n  # what lies behind the row in its last page
        for pos in range(last, -(-last // psize) * psize):
            c["k_pool"][int(tables[b, pos // psize]), :, pos % psize] = bad
            c["v_pool"][int(tables[b, pos // psize]), :, pos % psize] = bad
    used = {int(tables[b, p]) for b in range(len(nodes)) for p in range(-(-(contexts[b] + nodes[b]) // psize))}
    for page in set(range(c["k_pool"].shape[0])) - used:
        c["k_pool"][page] = bad
        c["v_pool"][page] = bad
    got = run_tree(c, device).cpu()
    dirty = torch.cat(dirty)
    assert torch.equal(got[~dirty], ref[~dirty])
    assert (~torch.isfinite(got[dirty].float())).any(dim=2).all()


def test_tree_attention_values_that_are_infinite_stay_so(device):
    """A token that sees an infinite V has it where its weight is not zero: inf with its sign, NaN only where both meet."""
    c = tree_case(8, [3], [40], 8, 2)
    pos = 41
    page, off = int(c["page_table"][0, pos // 16]), pos % 16
    c["masks"] = torch.tensor([[1], [2], [5]])
    c["v_pool"][page, :, off, 0] = math.inf
    c["v_pool"][page, :, off, 1] = -math.inf
    c["v_pool"][page, :, off, 2] = math.nan
    got = run_tree(c, device).cpu()
    assert (got[1, :, 0] == math.inf).all() and (got[1, :, 1] == -math.inf).all() and got[1, :, 2].isnan().all()
    assert torch.isfinite(got[1, :, 3:]).all() and torch.isfinite(got[0]).all() and torch.isfinite(got[2]).all()


@pytest.mark.parametrize("hq,hkv,d,dtype", KINDS)
def test_tree_attention_scores_without_a_finite_one(device, hq, hkv, d, dtype):
    """A token whose scores are all -inf gives NaN (a softmax over them), one that sees a finite one is not touched."""
    c = tree_case(6, [4], [0], hq, hkv, d=d, dtype=dtype)
    c["masks"] = torch.tensor([[1], [2], [3], [8]])
    c["q"] = c["q"].abs() + 0.5
    c["k_pool"] = c["k_pool"].abs() + 0.5
    page = int(c["page_table"][0, 0])
    c["k_pool"][page, :, 0] = -math.inf
    got = run_tree(c, device).cpu()
    assert got[0].isnan().all()
    v1 = c["v_pool"][page, :, 1].repeat_interleave(hq // hkv, dim=0)
    assert torch.equal(got[1], v1) and torch.equal(got[2], v1)
    assert torch.isfinite(got[3]).all()


@pytest.mark.parametrize("hq,hkv,d,dtype", KINDS)
def test_tree_attention_scores_that_rise_and_fall(device, hq, hkv, d, dtype):
    for factor in (40.0, -40.0):
        c = tree_case(11, [20, 3], [900, 2], hq, hkv, d=d, dtype=dtype)
        t = torch.arange(900)
        pages = c["page_table"][0].long()[t // 16]
        c["k_pool"][pages, :, t % 16] = (c["k_pool"][pages, :, t % 16].float() * 0.05 +
                                         (t / 900 * factor / d)[:, None, None]).to(dtype)
        c["q"] = (c["q"].float() * 0.1 + 1.0).to(dtype)
        check_tree(c, run_tree(c, device))


@pytest.mark.parametrize("hq,hkv,d,dtype", KINDS)
def test_tree_attention_leaves_other_rows(device, hq, hkv, d, dtype):
    """Query rows between and behind the counted ones, of rows that were not granted, keep what out held; their q and
    masks may be anything, and so may the table of a row without tokens."""
    c = tree_case(2, [5, 0, 9, 0], [60, 10, 0, 0], hq, hkv, d=d, dtype=dtype, gaps=[2, 4, 0, 3])
    ref, _ = attention64(c, d ** -0.5)
    dead = ref.isnan()
    c["q"][dead] = math.nan
    c["masks"][dead.any(dim=2).any(dim=1)] = -1
    c["page_table"][1] = 1 << 30
    c["page_table"][3] = -5
    c["seq_lens"][3] = 0
    out = torch.full(c["q"].shape, 7.0, dtype=dtype, device=device)
    got = run_tree(c, device, out=out)
    assert got is out
    check_tree(c, got)
    assert (got.cpu()[dead] == 7.0).all()


@pytest.mark.parametrize("hq,hkv,d,dtype", KINDS)
@pytest.mark.parametrize("nodes,words,context", [([5, 65, 64, 0, 9], 1, 0), ([300, 3], 2, 70), ([2, 257, 200, 600], 4, 3000)])
def test_tree_attention_rows_past_their_masks(device, hq, hkv, d, dtype, nodes, words, context):
    """A row of more tokens than its masks have bits for is refused: its tokens yield NaN (nothing says which drafted tokens
    they see, and the first ones are no context); other rows are as ever, and check_tables raises."""
    c = tree_case(len(nodes), nodes, [context + 3 * b for b in range(len(nodes))], hq, hkv, d=d, words=words, dtype=dtype,
                  gaps=[b % 2 for b in range(len(nodes))])
    over = [b for b, n in enumerate(nodes) if n > 64 * words]
    out = torch.full_like(c["q"], 7.0).to(device)
    got = run_tree(c, device, out=out).cpu()
    refused = torch.zeros(got.shape[0], dtype=torch.bool)
    for b in over:
        first = int(c["offsets"][b])
        refused[first: first + nodes[b]] = True
    assert got[refused].isnan().all()
    with pytest.raises(ValueError, match=f"row {over[0]}: counts exceed"):
        run_tree(c, device, check_tables=True)
    c["counts"][over] = 0
    ref, tol = attention64(c, d ** -0.5)
    idle = ref.isnan() & ~refused[:, None, None]
    assert (got[idle] == 7.0).all()
    live = ~ref.isnan()
    assert bool(((got.double() - ref).abs()[live] <= tol[live]).all())


@pytest.mark.parametrize("rows,nodes,hq,hkv", [(300, 3, 8, 2), (700, 1, 4, 4), (2300, 2, 4, 4), (40, 200, 8, 2)])
def test_tree_attention_many_rows(device, rows, nodes, hq, hkv):
    ns = [(nodes * (1 + b % 2)) if nodes < 200 else nodes for b in range(rows)]
    c = tree_case(rows, ns, [(37 * b) % 90 for b in range(rows)], hq, hkv, words=4)
    got = run_tree(c, device)
    some = sorted({0, 1, rows // 3, rows // 2, rows - 2, rows - 1})
    for b in some:
        lo, hi = int(c["offsets"][b]), int(c["offsets"][b + 1])
        one = dict(c, q=c["q"][lo:hi], masks=c["masks"][lo:hi], page_table=c["page_table"][b: b + 1],
                   seq_lens=c["seq_lens"][b: b + 1], offsets=i32([0, hi - lo]), counts=c["counts"][b: b + 1])
        check_tree(one, got[lo:hi])


def tree_heads64(c, scale):
    """attention64 for as many query as KV heads and one row, head by head in float64 on the tensors' device: (out,
    tolerance)."""
    q, length, n = c["q"].double(), int(c["seq_lens"][0]), c["q"].shape[0]
    t = torch.arange(length, device=q.device)
    pages, psize = c["page_table"][0].long()[t // c["k_pool"].shape[2]], c["k_pool"].shape[2]
    seen = torch.ones((n, length), dtype=torch.bool)
    seen[:, length - n:] = bits_of(c["masks"].cpu(), n)
    seen = seen.to(q.device)
    out, tol = torch.empty_like(q), torch.empty_like(q)
    for h in range(q.shape[1]):
        k, v = c["k_pool"][pages, h, t % psize].double(), c["v_pool"][pages, h, t % psize].double()
        s = (q[:, h] @ k.T * scale).masked_fill(~seen, -math.inf)
        e = torch.exp(s - s.max(dim=1, keepdim=True).values)
        l = e.sum(dim=1, keepdim=True)
        out[:, h] = e @ v / l
        off = 260 * U32 * abs(scale) * (q[:, h].abs() @ k.abs().T).max(dim=1, keepdim=True).values
        tol[:, h] = (e @ v.abs() / l) * (2 * U16 + 2 * off) + v.abs().sum(dim=0) * 2.0 ** -25 / l + U16 * out[:, h].abs()
    return out, tol


@pytest.mark.parametrize("heads,n,context", [
    (256, 2, 4500), (256, 100, 4600), (256, 200, 4433),  # one workgroup a head: 70 stages, pages of 64 of them at a time
    (1, 3, 9000), (1, 150, 17000),                       # 256 workgroups: a tile's pieces are more than 32
])
def test_tree_attention_long(device, heads, n, context):
    g = torch.Generator(device).manual_seed(n)
    pages = -(-(context + n) // 16)
    pool = lambda: torch.randn((pages + 3, heads, 16, 128), generator=g, dtype=torch.float16, device=device)
    c = dict(q=torch.randn((n, heads, 128), generator=g, dtype=torch.float16, device=device), k_pool=pool(), v_pool=pool(),
             page_table=torch.randperm(pages + 3, generator=g, device=device)[None, :pages].int(),
             seq_lens=i32([context + n]).to(device), offsets=i32([0, n]).to(device), counts=i32([n]).to(device),
             masks=mask_words(seen_sets(tree(n, 5, "any")), 4).to(device))
    ref, tol = tree_heads64(c, 128 ** -0.5)
    got = run_tree(c, device)
    assert bool(((got.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("hq,hkv,d,dtype", KINDS)
@pytest.mark.parametrize("nodes", [[3], [40], [64, 7]])
def test_tree_attention_of_huge_scores(device, hq, hkv, d, dtype, nodes):
    """Scores of up to 10^8 that are exact, 2^20 apart or equal: a token's answer is the mean of V over those of the greatest,
    off by the rounding of the weights (equal: they are 1, or 2^x with one x for all), of the sums and of the answer."""
    c = tree_case(21, nodes, [70] * len(nodes), hq, hkv, d=d, dtype=dtype)
    g = torch.Generator().manual_seed(2)
    steps = torch.randint(-90, 91, c["k_pool"].shape[:3], generator=g)
    c["k_pool"].zero_()
    c["k_pool"][..., 0] = steps.to(dtype)
    c["q"].zero_()
    c["q"][..., 0] = torch.tensor([1.0, -1.0])[torch.randint(0, 2, c["q"].shape[:2], generator=g)].to(dtype)
    got = run_tree(c, device, scale=2.0 ** 20).cpu().double()
    for b, n in enumerate(nodes):
        first, t = int(c["offsets"][b]), torch.arange(70 + n)
        pages = c["page_table"][b].long()[t // 16]
        for i in range(n):
            seen = torch.cat([torch.ones(70, dtype=torch.bool), bits_of(c["masks"][first + i: first + i + 1], n)[0]])
            for h in range(hq):
                s = steps[pages, h // (hq // hkv), t % 16] * float(c["q"][first + i, h, 0])
                best = (s == s[seen].max()) & seen
                v = c["v_pool"][pages[best], h // (hq // hkv), t[best] % 16].double()
                tol = (2 * U16 if dtype == torch.float16 else 100 * U32) * v.abs().mean(dim=0) + 2.0 ** -25
                assert bool(((got[first + i, h] - v.mean(dim=0)).abs() <= tol).all())


@pytest.mark.parametrize("d,dtype", [(128, torch.float16), (64, torch.float32)])
def test_tree_attention_far_in_the_pools(device, d, dtype):
    """Pages whose elements have numbers past 2^31: the same bits as from the start of small pools."""
    c = tree_case(13, [20, 3], [100, 40], 8, 2, d=d, dtype=dtype)
    want = run_tree(c, device)
    small = c["k_pool"].shape[0]
    slots = 2 ** 31 // (2 * 16 * d) + small
    pools = {}
    for name in ("k_pool", "v_pool"):
        pools[name] = torch.empty((slots, 2, 16, d), dtype=dtype, device=device)
        pools[name][-small:] = c[name].to(device)
    far = {**{k: v.to(device) for k, v in c.items()}, **pools}
    far["page_table"] = far["page_table"] + (slots - small)
    assert torch.equal(run_tree(far, device), want)


def test_tree_attention_chain_is_causal_prefill(device):
    from cacheir_amd import kernels

    c = {k: v.to(device) for k, v in tree_case(4, [33, 33], [70, 200], 32, 8, shape="chain").items()}
    a = kernels.paged_tree_attention(**c)
    b = kernels.paged_prefill_attention(c["q"], c["k_pool"], c["v_pool"], c["page_table"], c["seq_lens"], 33)
    assert (a.float() - b.float()).abs().max() <= 8 * U16  # (both within 4 u16 of values of about one)


@pytest.mark.parametrize("hq,hkv,d,dtype", KINDS)
def test_tree_attention_in_graphs_and_streams(device, hq, hkv, d, dtype):
    """A captured call follows lengths, counts, masks and tables between replays; two streams with a workspace each."""
    from cacheir_amd import kernels

    a = tree_case(21, [26, 3, 64], [300, 50, 0], hq, hkv, d=d, dtype=dtype)
    b = tree_case(22, [5, 64, 24], [17, 300, 200], hq, hkv, d=d, dtype=dtype, gaps=[0, 0, 0])
    b["k_pool"], b["v_pool"] = a["k_pool"], a["v_pool"]
    width = max(a["page_table"].shape[1], b["page_table"].shape[1])
    pad = lambda t: torch.nn.functional.pad(t, (0, width - t.shape[1]))
    a["page_table"], b["page_table"] = pad(a["page_table"]), pad(b["page_table"] % a["k_pool"].shape[0])
    assert a["q"].shape == b["q"].shape
    s = {k: v.to(device) for k, v in a.items()}
    out = torch.empty_like(s["q"])
    mk = lambda: kernels.tree_attention_workspace(s["q"].shape[0], 3, hq, hkv, d, 16, width, dtype, device)
    ws = mk()
    go = lambda: kernels.paged_tree_attention(**s, out=out, workspace=ws)
    go()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for c in (a, b, a, b):
        for k in s:
            s[k].copy_(c[k])
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        check_tree(c, replayed)
        assert torch.equal(go(), replayed)
    da, db = ({k: v.to(device) for k, v in c.items()} for c in (a, b))
    streams, wss = [torch.cuda.Stream(), torch.cuda.Stream()], [mk(), mk()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (c, st) in enumerate(zip((da, db), streams)):
            with torch.cuda.stream(st):
                got[i].append(kernels.paged_tree_attention(**c, workspace=wss[i]))
    torch.cuda.synchronize()
    for i, c in enumerate((a, b)):
        check_tree(c, got[i][0])
        assert all(torch.equal(got[i][0], g) for g in got[i])


def test_tree_attention_refusals(device):
    from cacheir_amd import kernels

    c = {k: v.to(device) for k, v in tree_case(1, [4, 3], [20, 0], 8, 2).items()}
    go = lambda **kw: kernels.paged_tree_attention(**{**c, **kw})
    for exc, match, kw in [
        (ValueError, "q must be", dict(q=c["q"][0])),
        (ValueError, "contiguous", dict(q=c["q"][:, ::2])),
        (TypeError, "share a dtype", dict(k_pool=c["k_pool"].float())),
        (ValueError, "v_pool|pools", dict(v_pool=c["v_pool"][:-1])),
        (TypeError, "int32", dict(offsets=c["offsets"].long())),
        (ValueError, "offsets", dict(offsets=c["offsets"][:-1])),
        (ValueError, "counts", dict(counts=c["counts"][:-1])),
        (ValueError, "masks", dict(masks=c["masks"][:-1])),
        (TypeError, "int64", dict(masks=c["masks"].int())),
        (RuntimeError, "words must be", dict(masks=c["masks"].repeat(1, 5))),
        (ValueError, "on the GPU", dict(q=c["q"].cpu())),
        (ValueError, "page_table", dict(page_table=c["page_table"].cpu())),
        (ValueError, "out must be", dict(out=torch.empty_like(c["q"][:-1]))),
        (RuntimeError, "workspace too small", dict(page_table=torch.nn.functional.pad(c["page_table"], (0, 600)),
                                                       workspace=torch.empty(4, dtype=torch.uint8, device=device))),
        (ValueError, "workspace", dict(workspace=torch.empty(4, dtype=torch.uint8))),
        (ValueError, "offsets must ascend", dict(offsets=i32([4, 0, 7]).to(device), check_tables=True)),
        (ValueError, "offsets must ascend", dict(offsets=i32([0, 4, 8]).to(device), check_tables=True)),
        (ValueError, "row 1: counts", dict(counts=i32([4, 4]).to(device), check_tables=True)),
        (ValueError, "outside the pool", dict(page_table=c["page_table"] + 99, check_tables=True)),
        (ValueError, "capacity", dict(seq_lens=c["seq_lens"] + 99, check_tables=True)),
    ]:
        with pytest.raises(exc, match=match):
            go(**kw)
    none = go(q=c["q"][:0], masks=c["masks"][:0], offsets=i32([0, 0, 0]).to(device))
    assert none.shape == (0, 8, 128)


# ------------------------------------------------------- norm and rotation -----
def turned64(x, w, eps, pos, freq, layout, factor):
    y = x.double()
    y = y / (y.square().mean(dim=2, keepdim=True) + eps).sqrt() * w.double()
    half = freq.numel()
    if layout == "interleaved":
        ia, ib = 2 * torch.arange(half), 2 * torch.arange(half) + 1
    else:
        ia, ib = torch.arange(half), torch.arange(half, 2 * half)
    angle = pos.double()[:, None] * freq[None, :]
    c, s = (angle.cos() * factor)[:, None, :], (angle.sin() * factor)[:, None, :]
    a, b = y[..., ia], y[..., ib]
    out, mag = y.clone(), y.abs()
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia] = mag[..., ib] = abs(factor) * (a.abs() + b.abs())
    return out, mag


@pytest.mark.parametrize("tokens,hq,hkv,d,rot,layout,dt,kvdt,wdt", [
    (1, 4, 2, 64, 64, "interleaved", torch.float32, torch.float32, torch.float32),
    (1, 32, 8, 128, 128, "half", torch.float16, torch.float16, torch.float16),
    (37, 28, 4, 128, 64, "half", torch.float16, torch.float16, torch.float32),
    (5, 16, 8, 96, 96, "interleaved", torch.float16, torch.float16, torch.float16),  # six items a head
    (9, 8, 8, 80, 40, "half", torch.float16, torch.float16, torch.float16),
    (6, 8, 1, 256, 256, "half", torch.float32, torch.float16, torch.float32),
    (130, 3, 1, 256, 2, "interleaved", torch.float16, torch.float32, torch.float16),
    (3, 2, 1, 254, 254, "half", torch.float32, torch.float32, torch.float16),        # 127 single pairs
    (4, 5, 5, 2, 2, "half", torch.float16, torch.float16, torch.float32),
    (3, 6, 3, 20, 0, "interleaved", torch.float32, torch.float32, torch.float32),
    (4, 0, 2, 64, 64, "half", torch.float16, torch.float16, torch.float16),          # no queries
    (700, 2, 2, 130, 36, "half", torch.float16, torch.float16, torch.float16),
])
def test_norm_rope_append(device, tokens, hq, hkv, d, rot, layout, dt, kvdt, wdt):
    from cacheir_amd import kernels

    g = torch.Generator().manual_seed(tokens * 31 + d)
    qkv = (3.0 * torch.randn((tokens, (hq + 2 * hkv) * d), generator=g)).to(dt)
    q, k, v = (x.unflatten(1, (-1, d)) if x.shape[1] else x.reshape(tokens, 0, d)
               for x in qkv.split([hq * d, hkv * d, hkv * d], dim=1))
    qw, kw = (1.0 + 0.3 * torch.randn((2, d), generator=g)).to(wdt)
    psize, eps, factor = 16, 1e-5, 1.25
    pages = -(-tokens // psize) + 2
    slots = torch.randperm(pages * psize, generator=g)[:tokens]
    dead = torch.zeros(tokens, dtype=torch.bool)
    if tokens > 3:
        slots[2], slots[3], dead[2:4] = -1, pages * psize, True
    pos = torch.randint(0, 200000, (tokens,), generator=g, dtype=torch.int32)
    freq = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) / max(1, rot // 2))
    on = lambda x: x.to(device)
    dq = on(qkv)
    gq, gk, gv = (x.unflatten(1, (-1, d)) if x.shape[1] else x.reshape(tokens, 0, d)
                  for x in dq.split([hq * d, hkv * d, hkv * d], dim=1))
    kp, vp = (torch.full((pages, hkv, psize, d), 9.0, dtype=kvdt, device=device) for _ in range(2))
    out = torch.full((tokens, hq, d), 5.0, dtype=dt, device=device)
    got = kernels.norm_rope_append(gq, gk, gv, on(qw), on(kw), eps, on(pos), on(slots), on(freq), kp, vp, layout=layout,
                                   factor=factor, out=out)
    assert got is out and torch.equal(dq.cpu(), qkv)
    u = {torch.float16: U16, torch.float32: U32}

    def near(have, x, w, dtype):
        ref, mag = turned64(x, w, eps, pos, freq, layout, factor)
        tol = (d / 2 + 22) * U32 * mag + u[dtype] * ref.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        err = (have.double() - ref).abs()
        assert bool((err <= tol)[~dead].all()), float((err - tol)[~dead].max())

    if hq:
        near(got.cpu(), q, qw, dt)
        assert (got.cpu()[dead] == 5.0).all()
    live = slots[~dead]
    flat = lambda pool: pool.cpu().transpose(1, 2).reshape(-1, hkv, d)
    have = torch.zeros((tokens, hkv, d), dtype=kvdt)
    have[~dead] = flat(kp)[live]
    near(have, k, kw, kvdt)
    assert torch.equal(flat(vp)[live], v[~dead].to(kvdt))
    rest = torch.ones(pages * psize, dtype=torch.bool)
    rest[live] = False
    assert (flat(kp)[rest] == 9.0).all() and (flat(vp)[rest] == 9.0).all()
    if hq:  # in place, q a view of the projection
        kernels.norm_rope_append(gq, gk, gv, on(qw), on(kw), eps, on(pos), on(slots), on(freq), kp, vp, layout=layout,
                                 factor=factor, out=gq)
        assert torch.equal(gq.cpu()[~dead], got.cpu()[~dead]) and torch.equal(gq.cpu()[dead], q[dead])


def test_norm_rope_append_far_in_the_pools(device):
    """Slots whose elements have numbers past 2^31: the bits of a small pool."""
    from cacheir_amd import kernels

    g = torch.Generator(device).manual_seed(6)
    q, k, v = (torch.randn((9, h, 128), generator=g, dtype=torch.float16, device=device) for h in (4, 2, 2))
    w = torch.ones(128, device=device)
    pos, freq = torch.arange(9, device=device, dtype=torch.int32), kernels.rope_frequencies(128, 10000.0, device=device)
    slots = torch.arange(9, device=device) * 5
    pages = 2 ** 31 // (2 * 16 * 128)
    small, far = ([torch.zeros((n, 2, 16, 128), dtype=torch.float16, device=device) for _ in range(2)] for n in (3, pages + 3))
    go = lambda pools, at: kernels.norm_rope_append(q, k, v, w, w, 1e-6, pos, at, freq, *pools)
    assert torch.equal(go(small, slots), go(far, slots + 16 * pages))
    for a, b in zip(small, far):
        assert torch.equal(a, b[pages:]) and not b[:pages].any()


def test_norm_rope_append_of_extreme_heads(device):
    """Heads of zeros, of the smallest and largest values, with NaN and infinities; eps 0 on a head of zeros gives NaN."""
    from cacheir_amd import kernels

    d = 128
    x = torch.randn((6, 1, d), generator=torch.Generator().manual_seed(0)).half()
    x[0] = 0
    x[1] = 6e-8
    x[2] = 65504
    x[3, 0, 5] = math.nan
    x[4, 0, 5] = math.inf
    w = torch.ones(d, dtype=torch.float16, device=device)
    pool = lambda: torch.zeros((1, 1, 16, d), dtype=torch.float16, device=device)
    z = torch.zeros(0, dtype=torch.float64, device=device)
    go = lambda eps: kernels.norm_rope_append(x.to(device), x.to(device), x.to(device), w, w, eps, i32([0] * 6).to(device),
                                              torch.arange(6, device=device), z, pool(), pool()).cpu()
    y = go(1e-6)
    assert (y[0] == 0).all() and (y[2].float() - 1.0).abs().max() <= U16 * 2 and y[3].isnan().all() and y[4, 0, 5].isnan()
    assert (y[1].float() - 6e-8 / math.sqrt(1e-6 + 3.6e-15)).abs().max() <= 1e-6 and torch.isfinite(y[5]).all()
    assert go(0.0)[0].isnan().all()


# ------------------------------------------------------------------ logits -----
def logits64(x, offsets, history, lens, prompts, drafts, masks, rep, pres, freq, bias_ids, bias, allowed):
    """(values, tolerance) in float64, plain loops over what occurs."""
    rows, vocab = x.shape
    out = x.double().clone()
    tol = torch.zeros_like(out)
    for b in range(len(offsets) - 1):
        for row in range(offsets[b], offsets[b + 1]):
            count, given = {}, set()
            if history is not None:
                for i, t in enumerate(history[b].tolist()[: max(0, int(lens[b]))]):
                    if 0 <= t < vocab:
                        if prompts is not None and i < int(prompts[b]):
                            given.add(t)
                        else:
                            count[t] = count.get(t, 0) + 1
            if drafts is not None:
                n = offsets[b + 1] - offsets[b]
                for k in range(min(n, 64 * masks.shape[1])):
                    t = int(drafts[offsets[b] + k])
                    if int(masks[row, k // 64]) >> (k % 64) & 1 and 0 <= t < vocab:
                        count[t] = count.get(t, 0) + 1
            extra = {}
            if bias_ids is not None:
                for t, v in zip(bias_ids[b].tolist(), bias[b].tolist()):
                    if 0 <= t < vocab:
                        extra[t] = v
            for t in set(count) | given | set(extra):
                y = float(x[row, t])
                size = 0.0
                if t in count or t in given:
                    r = 1.0 if rep is None else float(rep[b])
                    y = y / r if y > 0 else y * r
                c = count.get(t, 0)
                size += abs(y)
                if c:
                    f, p = (0.0 if z is None else float(z[b]) for z in (freq, pres))
                    y = y - f * c - p
                    size += abs(f * c) + abs(p)
                y += extra.get(t, 0.0)
                size += abs(extra.get(t, 0.0))
                out[row, t] = y
                tol[row, t] = 4 * U32 * size + (U16 * abs(y) + 2.0 ** -25 if x.dtype == torch.float16 else U32 * abs(y))
            if allowed is not None:
                v = torch.arange(vocab)
                ok = (allowed[row].long()[v // 32] >> (v % 32) & 1) != 0
                out[row, ~ok] = -math.inf
                tol[row, ~ok] = 0.0
    return out, tol


def logits_case(seed, nodes, vocab, width, dtype, words=1, biases=5, pad=0, masked=True, drafts=True):
    g = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    batch, rows = len(nodes), sum(nodes)
    offsets = [0]
    sets = []
    for b, n in enumerate(nodes):
        sets += seen_sets(tree(n, seed + b)) if n else []
        offsets.append(len(sets))
    pick = lambda *s: (vocab * torch.rand(s, generator=g) ** 3).long().clamp_(0, vocab - 1)
    hist = pick(batch, width)
    if width > 3:
        hist[:, 1], hist[:, 2] = -1, vocab  # no tokens
    lens = [rng.randint(0, width) for _ in nodes]
    ids = pick(batch, biases)
    if biases > 2:
        ids[:, -2] = ids[:, 0]  # listed twice: the later one counts
        ids[:, 1] = -1
    bits = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=g).int()
    if rows > 2:
        bits[1], bits[2] = -1, 0
    wide = (4.0 * torch.randn((rows, vocab + pad), generator=g)).to(dtype)
    return dict(logits=wide[:, :vocab], offsets=i32(offsets), history=hist, history_lens=i32(lens),
                prompt_lens=i32([rng.randint(0, n + 2) for n in lens]),
                drafts=pick(rows) if drafts else None, masks=mask_words(sets, words) if drafts else None,
                repetition=0.6 + torch.rand(batch, generator=g), presence=torch.rand(batch, generator=g) - 0.3,
                frequency=torch.rand(batch, generator=g) - 0.3, bias_ids=ids, bias=3.0 * torch.randn((batch, biases), generator=g),
                allowed=bits if masked else None)


def reference_logits(c):
    full = dict(history=None, history_lens=None, prompt_lens=None, drafts=None, masks=None, repetition=None, presence=None,
                frequency=None, bias_ids=None, bias=None, allowed=None)
    full.update(c)
    off = list(range(full["logits"].shape[0] + 1)) if full.get("offsets") is None else full["offsets"].tolist()
    return logits64(full["logits"], off, full["history"], full["history_lens"], full["prompt_lens"], full["drafts"],
                    full["masks"], full["repetition"], full["presence"], full["frequency"], full["bias_ids"], full["bias"],
                    full["allowed"])


def near_logits(got, ref, tol):
    got, inf = got.cpu().double(), ref == -math.inf
    assert torch.equal(got == -math.inf, inf)
    err = (got - ref).abs()[~inf]
    assert bool((err <= tol[~inf]).all()), float((err - tol[~inf]).max())


@pytest.mark.parametrize("nodes,vocab,width,dtype,words,pad", [
    ([1], 1024, 40, torch.float32, 1, 0), ([1, 1, 1], 1, 3, torch.float32, 1, 0), ([1] * 4, 33, 100, torch.float16, 1, 0),
    ([5, 1, 12], 8192, 300, torch.float32, 1, 0), ([70, 3], 8193, 50, torch.float16, 2, 0),
    ([64, 0, 33, 1], 16384, 1000, torch.float16, 1, 0), ([2, 9], 20001, 5000, torch.float32, 1, 3),
    ([3, 200], 1000, 64, torch.float32, 4, 0), ([4, 4], 24576, 10, torch.float16, 1, 8), ([3, 1], 16390, 7, torch.float16, 1, 2),
    ([64, 6], 152064, 300, torch.float32, 1, 0), ([100, 12], 152063, 3000, torch.float16, 2, 1),  # more than 32 MB
])
@pytest.mark.parametrize("in_place", [False, True])
def test_adjust_logits(device, nodes, vocab, width, dtype, words, pad, in_place):
    from cacheir_amd import kernels

    c = logits_case(vocab, nodes, vocab, width, dtype, words=words, pad=pad)
    ref, tol = reference_logits(c)
    wide = torch.full((sum(nodes), vocab + pad), 3.5, dtype=dtype, device=device)
    wide[:, :vocab] = c["logits"].to(device)
    d = {k: v.to(device) for k, v in c.items()}
    d["logits"] = wide[:, :vocab]
    got = kernels.adjust_logits(**d, out=d["logits"] if in_place else None)
    near_logits(got, ref, tol)
    if in_place:
        assert got is d["logits"] and (wide[:, vocab:] == 3.5).all()
    else:
        assert torch.equal(d["logits"].cpu(), c["logits"])


@pytest.mark.parametrize("leave", [["history", "history_lens", "prompt_lens"], ["prompt_lens"], ["drafts", "masks"],
                                   ["bias_ids", "bias"], ["allowed"], ["repetition"], ["presence", "frequency"],
                                   ["history", "history_lens", "prompt_lens", "drafts", "masks", "bias", "bias_ids",
                                    "repetition", "presence", "frequency"],
                                   ["history", "history_lens", "prompt_lens", "drafts", "masks", "bias", "bias_ids",
                                    "repetition", "presence", "frequency", "allowed"]])
@pytest.mark.parametrize("in_place", [False, True])
def test_adjust_logits_parts(device, leave, in_place):
    from cacheir_amd import kernels

    c = logits_case(7, [1, 6, 2], 9000, 500, torch.float32)
    c = {k: v for k, v in c.items() if k not in leave}
    ref, tol = reference_logits(c)
    d = {k: v.to(device) for k, v in c.items()}
    near_logits(kernels.adjust_logits(**d, out=d["logits"] if in_place else None), ref, tol)


def test_adjust_logits_a_row_each(device):
    """No offsets: row b is sequence b's.  Values that no rule names keep their bits, NaN and infinities among them; NaN
    that a mask forbids becomes -inf."""
    from cacheir_amd import kernels

    c = logits_case(3, [1] * 5, 4099, 60, torch.float32, drafts=False)
    for name in ("offsets", "drafts", "masks"):
        del c[name]
    c["logits"] = c["logits"].clone()
    c["logits"][:, 11::50] = math.nan
    c["logits"][:, 12::50] = math.inf
    c["logits"][:, 13::50] = -math.inf
    c["allowed"][0] = -1
    ref, _ = reference_logits(c)
    d = {k: v.to(device) for k, v in c.items()}
    got = kernels.adjust_logits(**d).cpu()
    assert torch.equal(got == -math.inf, ref == -math.inf) and torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got == math.inf, ref == math.inf)
    assert (got[2] == -math.inf).all()  # a mask without a bit


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("drafts", [False, True])
def test_adjust_logits_values_and_bits(device, dtype, in_place, drafts):
    """Every value that some rule names, in rows of their own and in rows of trees, and the bits of those that none names:
    NaN of any payload, infinities, negative zeros and numbers below the normal range among them."""
    from cacheir_amd import kernels

    c = logits_case(13, [7, 1, 30] if drafts else [1] * 9, 9001, 200, dtype, drafts=drafts)
    if not drafts:
        for name in ("offsets", "drafts", "masks"):
            del c[name]
    kind, odd = ((torch.int32, [0x7fc01234, 0x7f800001, -0x3fffff, 0x7f800000, -0x800000, -2 ** 31, 1, -2 ** 31 + 77])
                 if dtype == torch.float32 else
                 (torch.int16, [0x7e21, 0x7c01, -0x1ff, 0x7c00, -0x400, -2 ** 15, 1, -2 ** 15 + 77]))
    bits = c["logits"].contiguous().view(kind).clone()
    for i, x in enumerate(odd):
        bits[:, 11 + i:: 50] = x
    c["logits"] = bits.view(dtype)
    ref, tol = reference_logits(c)
    d = {k: v.to(device) for k, v in c.items()}
    got = kernels.adjust_logits(**d, out=d["logits"] if in_place else None).cpu()
    kept = (tol == 0) & (ref != -math.inf) | (bits == odd[4]) & (ref == -math.inf)  # (-inf stays so under every rule)
    kept |= ref.isnan() & ~tol.isnan()
    assert torch.equal(got.view(kind)[kept], bits[kept]) and int(kept.sum()) > got.numel() // 3
    finite = ref.isfinite()
    # Below 2^-126 fp32 numbers lie 2^-149 apart, so each of the four roundings that logits64 counts in relative terms (a
    # quotient or product, an FMA, two sums) may be off by half of that, 2^-150, instead.
    tol = tol + (4 * 2.0 ** -150 if dtype == torch.float32 else 0.0)
    assert bool(((got.double() - ref).abs()[finite] <= tol[finite]).all()) and int((finite & ~kept).sum()) > 100
    assert torch.equal(got == -math.inf, ref == -math.inf) and torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got == math.inf, ref == math.inf)


def test_adjust_logits_the_same_token_many_times(device):
    from cacheir_amd import kernels

    n = 50000
    x = torch.full((2, 100), 2.0, device=device)
    got = kernels.adjust_logits(x, history=torch.full((2, n), 7, device=device), history_lens=i32([n, 3]).to(device),
                                frequency=torch.tensor([2.0 ** -10, 1.0], device=device))
    want = torch.full((2, 100), 2.0)
    want[0, 7], want[1, 7] = 2.0 - n * 2.0 ** -10, -1.0
    assert torch.equal(got.cpu(), want)


def test_adjust_logits_leaves_other_rows(device):
    from cacheir_amd import kernels

    c = logits_case(4, [2, 3, 4], 600, 20, torch.float32)
    c["offsets"] = i32([1, 2, 2, 6])
    ref, tol = reference_logits(c)
    d = {k: v.to(device) for k, v in c.items()}
    out = torch.full((9, 600), 8.0, device=device)
    got = kernels.adjust_logits(**d, out=out)
    near_logits(got[1:6], ref[1:6], tol[1:6])
    assert (got[0] == 8.0).all() and (got[6:] == 8.0).all()


def test_adjust_logits_in_graphs(device):
    """A captured call follows its inputs between replays (out of place, so that each replay starts from the logits)."""
    from cacheir_amd import kernels

    a = logits_case(31, [3, 5], 20000, 400, torch.float16)
    b = logits_case(32, [4, 4], 20000, 400, torch.float16)
    s = {k: v.to(device) for k, v in a.items()}
    out = torch.empty_like(s["logits"])
    go = lambda: kernels.adjust_logits(**s, out=out)
    go()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for c in (a, b, a, b):
        for k in s:
            s[k].copy_(c[k])
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        near_logits(out, *reference_logits(c))
        replayed = out.clone()
        assert torch.equal(go(), replayed)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_adjust_logits_at_any_address(device, dtype):
    """Rows that begin one element behind a 16-byte boundary, of odd strides, and their out alike."""
    from cacheir_amd import kernels

    c = logits_case(41, [9, 2], 8201, 300, dtype, pad=4)
    ref, tol = reference_logits(c)
    wide = torch.full((11, 8201 + 4), 3.5, dtype=dtype, device=device)
    wide[:, 1: 8202] = c["logits"].to(device)
    d = {**{k: v.to(device) for k, v in c.items()}, "logits": wide[:, 1: 8202]}
    into = torch.full((11, 8201 + 6), 3.5, dtype=dtype, device=device)
    near_logits(kernels.adjust_logits(**d, out=into[:, 3: 8204]), ref, tol)
    assert (into[:, :3] == 3.5).all() and (into[:, 8204:] == 3.5).all()
    near_logits(kernels.adjust_logits(**d, out=d["logits"]), ref, tol)
    assert (wide[:, :1] == 3.5).all() and (wide[:, 8202:] == 3.5).all()


def test_adjust_logits_of_many_rows(device):
    """Logits of more than 2^31 elements, in place: the last rows as in a small call."""
    from cacheir_amd import kernels

    vocab, rows = 152064, 2 ** 31 // 152064 + 5
    x = torch.zeros((rows, vocab), dtype=torch.float16, device=device)
    g = torch.Generator(device).manual_seed(4)
    x[-4:] = torch.randn((4, vocab), generator=g, dtype=torch.float16, device=device)
    hist = torch.randint(0, vocab, (4, 50), generator=g, device=device)
    kw = dict(repetition=torch.full((4,), 1.5, device=device), frequency=torch.full((4,), 0.25, device=device))
    want = kernels.adjust_logits(x[-4:], history=hist, history_lens=i32([50] * 4).to(device), **kw)
    offsets = torch.tensor([0] + [rows - 4 + i for i in range(5)], device=device, dtype=torch.int32)  # (rows 0 .. : row 0's)
    full = lambda t: torch.cat([torch.ones((1, *t.shape[1:]), dtype=t.dtype, device=device), t])
    kernels.adjust_logits(x, offsets, history=full(hist), history_lens=i32([0] + [50] * 4).to(device),
                          **{k: full(v) for k, v in kw.items()}, out=x)
    assert torch.equal(x[-4:], want) and not x[:-4].any()


def test_adjust_logits_refusals(device):
    from cacheir_amd import kernels

    c = {k: v.to(device) for k, v in logits_case(1, [2, 3], 100, 8, torch.float32).items()}
    go = lambda **kw: kernels.adjust_logits(**{**c, **kw})
    for exc, match, kw in [
        (ValueError, "rows, vocab", dict(logits=c["logits"][0])),
        (ValueError, "contiguous rows", dict(logits=c["logits"].T)),
        (TypeError, "dtype", dict(logits=c["logits"].double(), out=None)),
        (ValueError, "on the GPU", dict(logits=c["logits"].cpu())),
        (TypeError, "offsets", dict(offsets=c["offsets"].long())),
        (ValueError, "history", dict(history=c["history"][:1])),
        (ValueError, "go together", dict(history=None)),
        (ValueError, "go together", dict(masks=None)),
        (ValueError, "go together", dict(bias=None)),
        (ValueError, "prompt_lens needs", dict(history=None, history_lens=None)),
        (ValueError, "drafts need", dict(offsets=None, history=None, history_lens=None, prompt_lens=None, repetition=None,
                                         presence=None, frequency=None, bias=None, bias_ids=None)),
        (ValueError, "allowed", dict(allowed=c["allowed"][:, :-1])),
        (ValueError, "out must be", dict(out=torch.empty((5, 99), device=device))),
    ]:
        with pytest.raises(exc, match=match):
            go(**kw)
    wide = torch.zeros(9, 100, device=device)
    with pytest.raises(RuntimeError, match="overlaps"):
        go(logits=wide[:5], out=wide[1:6])
    with pytest.raises(RuntimeError, match="overlaps"):
        go(logits=wide[:5], out=wide.view(-1)[: 5 * 101].as_strided((5, 100), (101, 1)))
    assert kernels.adjust_logits(c["logits"][:0]).shape == (0, 100)


# ------------------------------------------------------------------ accept -----
def accept_ref(c, most):
    parents, drafts, targets, lens, table = (c[k].tolist() for k in ("parents", "drafts", "targets", "seq_lens", "page_table"))
    offsets, counts, psize = c["offsets"].tolist(), c["counts"].tolist(), c["k_pools"].shape[3]
    kp, vp = c["k_pools"].clone(), c["v_pools"].clone()
    accepted, paths, tokens, ends = [], [], [], []
    for b, n in enumerate(counts):
        o, start = offsets[b], lens[b] - n
        path = [0] if n else []
        while path and len(path) < most:
            kids = [k for k in range(path[-1] + 1, n) if parents[o + k] == path[-1] and drafts[o + k] == targets[o + path[-1]]]
            if not kids:
                break
            path.append(kids[0])
        for i, k in enumerate(path):
            (pa, oa), (pb, ob) = ((table[b][(start + x) // psize], (start + x) % psize) for x in (k, i))
            kp[:, pb, :, ob] = c["k_pools"][:, pa, :, oa]
            vp[:, pb, :, ob] = c["v_pools"][:, pa, :, oa]
        accepted.append(len(path))
        paths.append(path + [-1] * (most - len(path)))
        tokens.append([targets[o + k] for k in path] + [-1] * (most - len(path)))
        ends.append(start + len(path))
    return accepted, paths, tokens, ends, kp, vp


def accept_case(seed, nodes, contexts, layers, hkv, d, psize, dtype, ids=3, gaps=None, shape="any"):
    """Few different tokens, so that paths are long and siblings often equal."""
    g = torch.Generator().manual_seed(seed)
    base = tree_case(seed, nodes, contexts, hkv, hkv, d=d, psize=psize, words=4, dtype=dtype, gaps=gaps, shape=shape)
    gaps = gaps or [0] * len(nodes)
    parents = [p for b, (n, gap) in enumerate(zip(nodes, gaps)) for p in tree(n, seed * 100 + b, shape) + [0] * gap]
    randint = lambda n: torch.randint(0, ids, (n,), generator=g)
    shape5 = (layers,) + tuple(base["k_pool"].shape)
    return dict(parents=i32(parents), drafts=randint(len(parents)), targets=randint(len(parents)), seq_lens=base["seq_lens"],
                offsets=base["offsets"], counts=base["counts"], page_table=base["page_table"],
                k_pools=torch.randn(shape5, generator=g).to(dtype), v_pools=torch.randn(shape5, generator=g).to(dtype))


@pytest.mark.parametrize("nodes,contexts,layers,hkv,d,psize,dtype,most,ids", [
    ([1], [0], 1, 1, 64, 16, torch.float32, 1, 3), ([26, 0, 9, 64], [90, 5, 0, 31], 4, 2, 64, 16, torch.float32, 8, 3),
    ([200, 256, 3], [1, 100, 15], 2, 8, 128, 16, torch.float16, 256, 1), ([40] * 6, list(range(10, 16)), 3, 4, 96, 32, torch.float16, 12, 2),
    ([30, 17], [7, 50], 2, 3, 5, 7, torch.float16, 20, 2), ([30, 17], [7, 50], 2, 3, 7, 1, torch.float32, 20, 2),
    ([100, 64], [0, 9], 0, 1, 64, 16, torch.float16, 5, 2)])
@pytest.mark.parametrize("shape", ["any", "chain", "forest"])
def test_accept_drafts(device, nodes, contexts, layers, hkv, d, psize, dtype, most, ids, shape):
    from cacheir_amd import kernels

    c = accept_case(d + most, nodes, contexts, layers, hkv, d, psize, dtype, ids, gaps=[b % 3 for b in range(len(nodes))],
                    shape=shape)
    accepted, paths, tokens, ends, kp, vp = accept_ref(c, most)
    s = {k: v.to(device) for k, v in c.items()}
    got = kernels.accept_drafts(**s, most=most)
    assert got.accepted.tolist() == accepted and got.path.tolist() == paths
    assert got.tokens.tolist() == tokens and got.seq_lens.tolist() == ends
    assert torch.equal(s["k_pools"].cpu(), kp) and torch.equal(s["v_pools"].cpu(), vp)
    assert torch.equal(s["seq_lens"].cpu(), c["seq_lens"])


@pytest.mark.parametrize("shape,ids,most", [("any", 2, 256), ("any", 1, 256), ("chain", 1, 256), ("forest", 2, 9)])
@pytest.mark.parametrize("give_back", [False, True])
def test_accept_drafts_of_rows_past_256_tokens(device, shape, ids, most, give_back):
    """The context ends before all of a row's drafted tokens; those past the first 256 are never taken."""
    from cacheir_amd import kernels

    nodes, contexts, psize = [300, 5, 257, 1000, 256], [37, 9, 0, 130, 16], 16
    c = accept_case(91, nodes, contexts, 2, 2, 64, psize, torch.float16, ids, gaps=[0, 2, 0, 1, 0], shape=shape)
    ref = dict(c, parents=c["parents"].clone())
    for first, n in zip(c["offsets"].tolist(), nodes):
        ref["parents"][first + 256: first + max(n, 256)] = -1  # (accept_ref takes tokens by their parents)
    accepted, paths, tokens, ends, kp, vp = accept_ref(ref, most)
    s = {k: v.to(device) for k, v in c.items()}
    kw, back = {}, []
    if give_back:
        for b, (end, length) in enumerate(zip(ends, c["seq_lens"].tolist())):
            back += c["page_table"][b, -(-end // psize): -(-length // psize)].tolist()
        kw = dict(free_slots=torch.zeros(len(back) + 5, dtype=torch.int32, device=device),
                  free_head=i32([len(back) + 2]).to(device),
                  out=kernels.AcceptedDrafts.empty(len(nodes), most, device)._replace(seq_lens=s["seq_lens"]))
    got = kernels.accept_drafts(**s, most=most, **kw)
    assert got.accepted.tolist() == accepted and got.path.tolist() == paths and got.tokens.tolist() == tokens
    assert got.seq_lens.tolist() == ends
    assert torch.equal(s["k_pools"].cpu(), kp) and torch.equal(s["v_pools"].cpu(), vp)
    if give_back:
        assert kw["free_head"].item() == 2 and kw["free_slots"].tolist() == [0, 0] + back + [0] * 3


def test_accept_drafts_far_in_the_pools(device):
    """Layers of more than 2^32 bytes: what moves is where it belongs, and nothing else is written."""
    from cacheir_amd import kernels

    c = accept_case(51, [40, 9], [30, 3], 2, 2, 64, 16, torch.float32, ids=2, shape="chain")
    _, _, _, _, kp, vp = accept_ref(c, 256)
    small = c["k_pools"].shape[1]
    slots = 2 ** 30 // (2 * 16 * 64) + small
    s = {k: v.to(device) for k, v in c.items()}
    s["page_table"] = s["page_table"] + (slots - small)
    for name in ("k_pools", "v_pools"):
        s[name] = torch.zeros((2, slots, 2, 16, 64), device=device)
        s[name][:, -small:] = c[name].to(device)
    kernels.accept_drafts(**s, most=256)
    for name, want in (("k_pools", kp), ("v_pools", vp)):
        assert torch.equal(s[name][:, -small:].cpu(), want) and not s[name][:, :-small].any()


def test_accept_drafts_gives_pages_back(device):
    from cacheir_amd import kernels

    rows = 300  # more than the threads that scan them
    nodes = [(7 * b) % 40 for b in range(rows)]
    c = accept_case(77, nodes, [(5 * b) % 23 for b in range(rows)], 1, 1, 8, 4, torch.float32, 2)
    accepted, _, _, ends, kp, _ = accept_ref(c, 256)
    back = []
    for b, (end, length) in enumerate(zip(ends, c["seq_lens"].tolist())):
        back += c["page_table"][b, -(-end // 4): -(-length // 4)].tolist()
    head = len(back) + 3
    free = torch.arange(1000, 1000 + head + 5, dtype=torch.int32)
    want = torch.cat([free[:3], i32(back), free[head:]])
    s = {k: v.to(device) for k, v in c.items()}
    f, h = free.to(device), i32([head]).to(device)
    out = kernels.AcceptedDrafts.empty(rows, 256, device)._replace(seq_lens=s["seq_lens"])  # lengths in place
    got = kernels.accept_drafts(**s, most=256, free_slots=f, free_head=h, out=out)
    assert got.accepted.tolist() == accepted and s["seq_lens"].tolist() == ends and torch.equal(s["k_pools"].cpu(), kp)
    assert h.item() == 3 and torch.equal(f.cpu(), want)
    s = {k: v.to(device) for k, v in c.items()}  # a head that cannot take them: nothing is given back
    f, h = free.to(device), i32([len(back) - 1]).to(device)
    got = kernels.accept_drafts(**s, most=256, free_slots=f, free_head=h)
    assert h.item() == len(back) - 1 and torch.equal(f.cpu(), free) and got.seq_lens.tolist() == ends


def test_accept_drafts_refusals(device):
    from cacheir_amd import kernels

    c = {k: v.to(device) for k, v in accept_case(1, [3, 4], [5, 0], 2, 2, 64, 16, torch.float32).items()}
    go = lambda most=4, **kw: kernels.accept_drafts(**{**c, **kw}, most=most)
    both = torch.zeros((3,) + tuple(c["k_pools"].shape[1:]), device=device)
    for exc, match, kw in [
        (ValueError, "most must be", dict(most=0)), (ValueError, "most must be", dict(most=257)),
        (TypeError, "drafts", dict(drafts=c["drafts"].int())), (ValueError, "targets", dict(targets=c["targets"][:-1])),
        (ValueError, "counts", dict(counts=c["counts"][:-1])), (TypeError, "v_pools", dict(v_pools=c["v_pools"].half())),
        (ValueError, "pools must be", dict(k_pools=c["k_pools"][0])), (ValueError, "go together", dict(free_head=c["counts"][:1])),
        (RuntimeError, "overlap", dict(k_pools=both[:2], v_pools=both[1:])),
        (TypeError, "dtype", dict(k_pools=c["k_pools"].double(), v_pools=c["v_pools"].double())),
    ]:
        with pytest.raises(exc, match=match):
            go(**kw)


# ------------------------------------------------------------- a run of them ---
def test_a_run_of_steps(device):
    """Steps of a server that drafts trees: page tables, masks, norm + rotary append, attention, logits, the model's
    choices, acceptance, pages given back; captured once and replayed, against the plain forms on the host after each."""
    from cacheir_amd import kernels

    batch, hq, hkv, d, psize, n, vocab, most, layers = 3, 8, 2, 128, 16, 12, 500, 6, 2
    g = torch.Generator().manual_seed(40)
    randn = lambda *s: torch.randn(s, generator=g).to(device)
    total, width = 120, 20
    pools = [torch.zeros((layers, total, hkv, psize, d), dtype=torch.float16, device=device) for _ in range(2)]
    table = torch.zeros((batch, width), dtype=torch.int32, device=device)
    free = torch.randperm(total, generator=g).int().to(device)
    head, lens = i32([0]).to(device), i32([0] * batch).to(device)
    parents_row = tree(n, 5)
    tokens = batch * n
    parents = i32(parents_row * batch).to(device)
    new = i32([n] * batch).to(device)
    t = kernels.StepTables.empty(batch, tokens, device)._replace(seq_lens=lens, free_head=head)
    dt = kernels.DraftTree(torch.empty((tokens, 1), dtype=torch.int64, device=device),
                           torch.empty(tokens, dtype=torch.int32, device=device))
    acc = kernels.AcceptedDrafts.empty(batch, most, device)._replace(seq_lens=lens)
    freq = kernels.rope_frequencies(d, 10000.0, device=device)
    drafts = torch.zeros(tokens, dtype=torch.int64, device=device)
    emb, wqkv, head_w = randn(vocab, 64), randn(layers, 64, (hq + 2 * hkv) * d) / 8, randn(hq * d, vocab) / 30
    qw, kw = 1 + 0.1 * randn(d), 1 + 0.1 * randn(d)
    history = torch.zeros((batch, 400), dtype=torch.int64, device=device)
    rep, freqs = torch.full((batch,), 1.3, device=device), torch.full((batch,), 0.1, device=device)
    keep = {}

    def step():
        kernels.extend_page_tables(table, lens, new, free, head, page_size=psize, max_tokens=tokens, out=t)
        kernels.draft_tree(parents, lens, t.offsets, t.granted, words=1, out=dt)
        x = emb[drafts]
        for layer in range(layers):
            q, k, v = (y.unflatten(1, (-1, d)) for y in (x @ wqkv[layer]).half().split([hq * d, hkv * d, hkv * d], dim=1))
            q = kernels.norm_rope_append(q, k, v, qw, kw, 1e-6, dt.positions, t.slot_map, freq, pools[0][layer],
                                         pools[1][layer], layout="half")
            o = kernels.paged_tree_attention(q, pools[0][layer], pools[1][layer], table, lens, t.offsets, t.granted, dt.masks)
            keep["q", layer], keep["o", layer] = q, o
            x = x + o.view(tokens, hq * d).float()[:, :64]
        logits = o.view(tokens, hq * d).float() @ head_w
        keep["raw"], keep["lens"], keep["masks"] = logits, lens.clone(), dt.masks.clone()
        keep["pools"] = [p.clone() for p in pools]
        adjusted = kernels.adjust_logits(logits, t.offsets, history=history, history_lens=lens - t.granted, drafts=drafts,
                                         masks=dt.masks, repetition=rep, frequency=freqs)
        keep["adjusted"] = adjusted
        keep["targets"] = kernels.argmax(adjusted)
        kernels.accept_drafts(parents, drafts, keep["targets"], lens, t.offsets, t.granted, table, *pools, most=most,
                              free_slots=free, free_head=head, out=acc)

    rng = random.Random(1)
    said = [[0] for _ in range(batch)]  # the token that opens the next tree is the last one

    def load():
        """Drafts of the next step: some confirmed by the run before it (guessed), the rest by chance."""
        rows = []
        for b in range(batch):
            rows += [said[b][-1]] + [rng.randrange(vocab) for _ in range(n - 1)]
            history[b, : len(said[b]) - 1] = torch.tensor(said[b][:-1], dtype=torch.int64)
        drafts.copy_(torch.tensor(rows))

    def probe_and_confirm(run):
        """Runs the step, then sets tokens along a path to what the model chose there, and runs it again from the same
        state: a step whose drafts are confirmed in part."""
        saved = [x.clone() for x in (table, free, head, lens, *pools)]
        run()
        torch.cuda.synchronize()
        d0 = drafts.clone()
        for b in range(batch):
            at, hops = 0, rng.randint(0, 3)
            for _ in range(hops):
                kids = [k for k in range(n) if parents_row[k] == at]
                if not kids:
                    break
                k = rng.choice(kids)
                d0[b * n + k] = keep["targets"][b * n + at]
                at = k
        for x, y in zip((table, free, head, lens, *pools), saved):
            x.copy_(y)
        drafts.copy_(d0)
        run()
        torch.cuda.synchronize()

    def check(before):
        lens0 = before
        grown = keep["lens"].tolist()
        assert grown == [a + n for a in lens0]
        sets = seen_sets(parents_row)
        assert torch.equal(keep["masks"].cpu(), mask_words(sets * batch, 1))
        for layer in range(layers):
            c = dict(q=keep["q", layer].cpu(), k_pool=keep["pools"][0][layer].cpu(), v_pool=keep["pools"][1][layer].cpu(),
                     page_table=table.cpu(), seq_lens=i32(grown), offsets=t.offsets.cpu(), counts=i32([n] * batch),
                     masks=keep["masks"].cpu())
            check_tree(c, keep["o", layer])
        ref, tol = reference_logits(dict(logits=keep["raw"].cpu(), offsets=t.offsets.cpu(), history=history.cpu(),
                                         history_lens=i32(lens0), drafts=drafts.cpu(), masks=keep["masks"].cpu(),
                                         repetition=rep.cpu(), frequency=freqs.cpu()))
        near_logits(keep["adjusted"], ref, tol)
        c = dict(parents=parents.cpu(), drafts=drafts.cpu(), targets=keep["targets"].cpu(), seq_lens=i32(grown),
                 offsets=t.offsets.cpu(), counts=i32([n] * batch), page_table=table.cpu(), k_pools=keep["pools"][0].cpu(),
                 v_pools=keep["pools"][1].cpu())
        accepted, paths, toks, ends, kp, vp = accept_ref(c, most)
        assert acc.accepted.tolist() == accepted and acc.path.tolist() == paths and acc.tokens.tolist() == toks
        assert lens.tolist() == ends and torch.equal(pools[0].cpu(), kp) and torch.equal(pools[1].cpu(), vp)
        held = [x for b in range(batch) for x in table[b, : -(-ends[b] // psize)].tolist()]
        assert sorted(held + free[int(head):].tolist()) == list(range(total))  # every page is somewhere, once
        for b in range(batch):
            said[b] += toks[b][: accepted[b]]
        return accepted

    load()
    before, longest = lens.tolist(), 0
    probe_and_confirm(step)
    check(before)
    load()
    state = [x.clone() for x in (table, free, head, lens, *pools)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for x, y in zip((table, free, head, lens, *pools), state):
        x.copy_(y)
    for _ in range(5):
        before = lens.tolist()
        load()
        probe_and_confirm(graph.replay)
        longest = max(longest, *check(before))
    assert longest > 1
