"""The operators of a serving step over shared prefixes, against plain 64-bit implementations on the CPU: page tables and
slot maps, rotary append, decode attention over shared prefixes, token log probabilities, and a run of them together.

Tolerances are sums of the roundings that the kernels make (u16 = 2^-11 and u32 = 2^-24: half a step of fp16 and fp32,
relative to the value):
* attention: each weight is rounded to fp16 once and the sum takes the rounded ones (2 u16 of sum w |v|, or 2^-25 / l per
  token for weights below fp16's normal range), scores are fp32 sums of 128 exact products (an exponent off by
  130 u32 |scale| sum |q k|, twice), the output is rounded to fp16 once more (u16 |out|);
* rotary: the reduced angle is rounded to fp32 (pi u32) and sine and cosine are good to 4 u32: 8 u32 factor (|a| + |b|),
  plus two fp32 roundings of the products and the rounding to the output type;
* log probabilities: fp32 sums of one lane's share (vocab / 256 + 100 additions, u32 each, and 4 u32 per exponential),
  plus the roundings of x - m and of the result.
Page tables, slots, positions and token ids are exact.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U16, U32 = 2.0 ** -11, 2.0 ** -24


# ------------------------------------------------------------------ attention --
def attention64(q, kp, vp, table, lens, scale):
    """(out, tolerance) in float64 from CPU tensors of any dtype."""
    batch, hq, d = q.shape
    hkv, psize = kp.shape[1], kp.shape[2]
    fp16 = q.dtype == torch.float16
    q, kp, vp = q.double(), kp.double(), vp.double()
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(batch):
        n = min(int(lens[b]), table.shape[1] * psize)
        if n <= 0:
            continue
        t = torch.arange(n)
        pages = table[b].long()[t // psize]
        for h in range(hkv):
            g = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            k, v = kp[pages, h, t % psize], vp[pages, h, t % psize]
            s = q[b, g] @ k.T * scale
            e = torch.exp(s - s.max(dim=1, keepdim=True).values)
            l = e.sum(dim=1, keepdim=True)
            w = e / l
            out[b, g] = w @ v
            off = 260 * U32 * abs(scale) * (q[b, g].abs() @ k.abs().T).max(dim=1, keepdim=True).values
            mass = w @ v.abs()
            tol[b, g] = mass * (2 * U16 + 2 * off) + v.abs().sum(dim=0) * 2.0 ** -25 / l + U16 * out[b, g].abs()
            if not fp16:
                tol[b, g] = mass * (2 * off + (n + 64) * U32) + 2 * U32 * out[b, g].abs()
    return out, tol


def shared_case(seed, groups, suffix, hq, hkv, psize=16, d=128, dtype=torch.float16, short=(), extra=3):
    """Groups of (rows, prefix tokens): page tables whose rows share the whole pages of their prefix; row b holds its
    prefix and suffix[b] tokens, rows in ``short`` (row -> length) something else.  CPU tensors."""
    g = torch.Generator().manual_seed(seed)
    rows, lens, used, b = [], [], 0, 0
    for n, prefix in groups:
        whole = prefix // psize
        common = list(range(used, used + whole))
        used += whole
        for _ in range(n):
            length = prefix + suffix[b]
            own = -(-length // psize) - whole
            rows.append(common + list(range(used, used + own)))
            used += own
            lens.append(dict(short).get(b, length))
            b += 1
    width = max(len(r) for r in rows) + 1
    perm = torch.randperm(used + extra, generator=g)
    table = torch.zeros((len(rows), width), dtype=torch.int32)
    for i, r in enumerate(rows):
        table[i, : len(r)] = perm[torch.tensor(r, dtype=torch.long)].int()
    randn = lambda *s: torch.randn(s, generator=g).to(dtype)
    kp, vp = randn(used + extra, hkv, psize, d), randn(used + extra, hkv, psize, d)
    first = np.cumsum([0] + [n for n, _ in groups])
    return dict(q=randn(len(rows), hq, d), k_pool=kp, v_pool=vp, page_table=table,
                seq_lens=torch.tensor(lens, dtype=torch.int32), group_rows=torch.tensor(first, dtype=torch.int32),
                prefix_lens=torch.tensor([p // psize * psize for _, p in groups], dtype=torch.int32))


def run_shared(case, device, scale=None, **kw):
    from cacheir_amd import kernels

    return kernels.paged_decode_attention_shared(**{k: v.to(device) for k, v in case.items()}, scale=scale, **kw)


def check_shared(case, got, scale=None):
    scale = case["q"].shape[2] ** -0.5 if scale is None else scale
    ref, tol = attention64(case["q"], case["k_pool"], case["v_pool"], case["page_table"], case["seq_lens"], scale)
    err = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got).all()
    assert bool((err <= tol).all()), f"max excess {(err - tol).max():.3e}, max error {err.max():.3e}"


@pytest.mark.parametrize("hq,hkv,groups,suffix,psize", [
    (8, 2, [(1, 0)], [1], 16),                               # one row, one token
    (32, 8, [(4, 500)], [1, 40, 17, 16], 16),                # one tile of 16 vectors, a prefix that ends inside a page
    (28, 4, [(9, 96)], [3] * 9, 16),                         # 63 vectors
    (32, 8, [(40, 1024)], list(range(1, 41)), 16),           # 160 vectors: a whole tile and one of 32
    (16, 1, [(17, 640)], [5] * 17, 32),                      # one KV head, 16 query heads each
    (32, 1, [(3, 288)], [40, 1, 100], 48),                   # 32 query heads, pages of three tiles
    (8, 8, [(5, 64), (1, 333), (7, 0), (2, 2000)], list(range(3, 18)), 16),
    (4, 4, [(3, 31), (3, 32), (3, 33)], [1, 2, 33, 31, 32, 64, 1, 1, 1], 64),
])
def test_shared_attention_shapes(device, hq, hkv, groups, suffix, psize):
    case = shared_case(hq + len(suffix), groups, suffix, hq, hkv, psize)
    check_shared(case, run_shared(case, device, check_tables=True))


@pytest.mark.parametrize("psize,whole,prefixes", [
    (64, [64, 128, 192, 640], [32, 100, 191, 577]), (48, [48, 96, 144, 480], [47, 95, 97, 479]),
    (16, [16, 32, 48, 640], [1, 31, 33, 639]), (128, [128, 128, 256, 640], [33, 127, 160, 600])])
@pytest.mark.parametrize("rows,hq,hkv", [(3, 8, 2), (20, 16, 2)])
def test_shared_attention_prefixes_that_end_inside_a_page(device, psize, whole, prefixes, rows, hq, hkv):
    """Prefixes that are no whole number of pages, of 32-token blocks or of either, the last page common to the rows (what
    follows the prefix in it is theirs too); some rows end inside the prefix or that page."""
    case = shared_case(17, [(rows, p) for p in whole], [(13 * b) % 70 for b in range(4 * rows)], hq, hkv, psize)
    case["prefix_lens"] = torch.tensor(prefixes, dtype=torch.int32)
    for g, p in enumerate(prefixes):
        case["seq_lens"][g * rows + 1] = p
        case["seq_lens"][g * rows + 2] = p - 1
    check_shared(case, run_shared(case, device, check_tables=True))
    case["page_table"][1, 0] = case["page_table"][1, 0] + (1 if case["page_table"][1, 0] == 0 else -1)
    with pytest.raises(ValueError, match="group 0: rows with other pages"):
        run_shared(case, device, check_tables=True)


@pytest.mark.parametrize("seed", range(8))
def test_shared_attention_random_groups(device, seed):
    rng = np.random.default_rng(seed)
    hq, hkv = [(32, 8), (28, 4), (16, 8), (6, 2)][seed % 4]
    n = int(rng.integers(1, 6))
    prefix = lambda: int(rng.choice([0, rng.integers(1, 200), rng.integers(200, 1500)]))
    groups = [(int(rng.integers(1, 30)), prefix()) for _ in range(n)]
    rows = sum(r for r, _ in groups)
    suffix = [int(x) for x in rng.integers(0, int(rng.choice([3, 40, 400])), rows)]
    short = {int(b): int(rng.integers(0, 40)) for b in rng.choice(rows, rows // 6, replace=False)}
    case = shared_case(seed, groups, suffix, hq, hkv, int(rng.choice([16, 32])), short=short)
    scale = float(rng.choice([128 ** -0.5, -0.3, 0.0, 1.0]))
    check_shared(case, run_shared(case, device, scale=scale), scale)


def test_shared_attention_many_rows_and_long_context(device):
    """More rows than threads of a workgroup; one sequence long enough for every workgroup."""
    case = shared_case(3, [(700, 64), (1, 0)], [int(x) for x in np.random.default_rng(1).integers(0, 9, 701)], 4, 2)
    check_shared(case, run_shared(case, device))
    case = shared_case(4, [(2, 20000)], [9000, 3], 4, 1)
    check_shared(case, run_shared(case, device))


def test_shared_attention_rows_at_the_edges(device):
    """Lengths 0 and past the table, rows shorter than their prefix (the first one too), rows outside every group, groups
    out of order (nothing is shared then), empty groups: the attention of each row alone."""
    case = shared_case(5, [(6, 320), (4, 160)], [7, 0, 30, 1, 2, 3, 9, 9, 9, 9], 8, 2,
                       short={1: 0, 2: 100, 3: 320, 4: 319})
    check_shared(case, run_shared(case, device))
    check_shared(case | {"seq_lens": case["seq_lens"].clone().index_fill_(0, torch.tensor([0]), 50)}, run_shared(
        case | {"seq_lens": case["seq_lens"].clone().index_fill_(0, torch.tensor([0]), 50)}, device))
    long = case["seq_lens"].clone()
    long[5] = 10 ** 6  # clamped to the table
    check_shared(case | {"seq_lens": long}, run_shared(case | {"seq_lens": long}, device))
    for rows, prefix in ([[2, 6], [320]], [[6, 2, 10], [320, 160]], [[0, 6, 6, 6, 10], [320, 5, 10 ** 9, 160]],
                         [[0, 20], [320]], [[-1, 6], [320]], [[0], []], [[0, 6, 10], [-5, 0]]):
        c = case | {"group_rows": torch.tensor(rows, dtype=torch.int32),
                    "prefix_lens": torch.tensor(prefix, dtype=torch.int32)}
        check_shared(c, run_shared(c, device))


@pytest.mark.parametrize("dtype,d,psize,hq,hkv", [
    (torch.float32, 64, 16, 4, 2), (torch.float32, 128, 16, 8, 2), (torch.float16, 64, 16, 4, 2),
    (torch.float16, 128, 8, 8, 2), (torch.float16, 128, 16, 33, 1)])
def test_shared_attention_sizes_that_read_each_row_alone(device, dtype, d, psize, hq, hkv):
    case = shared_case(6, [(3, 96), (2, 50)], [1, 200, 17, 3, 4], hq, hkv, psize, d, dtype)
    check_shared(case, run_shared(case, device))


@pytest.mark.parametrize("rows,groups", [(2048, 256), (2049, 200), (514, 257)])
def test_shared_attention_at_the_limits_of_rows_and_groups(device, rows, groups):
    """The most rows and groups that share, and one more of each (every row alone)."""
    sizes = [rows // groups + (g < rows % groups) for g in range(groups)]
    case = shared_case(18, [(n, 32 * (g % 4)) for g, n in enumerate(sizes)], [b % 37 for b in range(rows)], 2, 1)
    check_shared(case, run_shared(case, device, check_tables=True))


def test_shared_attention_pools_off_16_bytes(device):
    case = shared_case(7, [(3, 96)], [1, 20, 17], 8, 2)
    dev = {k: v.to(device) for k, v in case.items()}
    for name in ("k_pool", "v_pool"):
        t = dev[name]
        raw = torch.empty(t.numel() + 4, dtype=t.dtype, device=device)
        dev[name] = raw[4:].view(t.shape).copy_(t)
    from cacheir_amd import kernels

    check_shared(case, kernels.paged_decode_attention_shared(**dev))


def test_shared_attention_q_and_out_off_their_alignment(device):
    """q off 16 bytes or out off 8 (the rows of a larger buffer): each row alone."""
    case = shared_case(7, [(3, 96)], [1, 20, 17], 8, 2)
    dev = {k: v.to(device) for k, v in case.items()}
    from cacheir_amd import kernels

    raw = torch.empty(dev["q"].numel() + 4, dtype=torch.float16, device=device)
    check_shared(case, kernels.paged_decode_attention_shared(**(dev | {"q": raw[4:].view(dev["q"].shape).copy_(dev["q"])})))
    raw = torch.empty(dev["q"].numel() + 2, dtype=torch.float16, device=device)
    check_shared(case, kernels.paged_decode_attention_shared(**dev, out=raw[2:].view(dev["q"].shape)))


def test_shared_attention_scores_at_the_limits(device):
    """Scores past 2^24, keys that make every score -inf (NaN), and infinities behind the last token (which stay out)."""
    case = shared_case(8, [(5, 128), (2, 0)], [5, 1, 40, 33, 70, 20, 64], 8, 2)
    case["q"][:, 1] *= 3000.0
    case["k_pool"][:, 0] *= 500.0
    got = run_shared(case, device, scale=20.0).cpu()
    q, kp = case["q"].double(), case["k_pool"].double()
    assert torch.isfinite(got).all()
    for b in (0, 3, 6):  # one weight is 1, the rest 0: the value of the best token
        n = int(case["seq_lens"][b])
        t = torch.arange(n)
        pages = case["page_table"][b].long()[t // 16]
        s = kp[pages, 0, t % 16] @ q[b, 1] * 20.0
        top = s.topk(2).values
        assert top[0] - top[1] > 2.0 ** 10
        assert torch.equal(got[b, 1], case["v_pool"][pages, 0, t % 16][s.argmax()])
    case = shared_case(9, [(5, 128), (2, 0)], [5, 1, 40, 33, 70, 20, 64], 8, 2)
    clean = run_shared(case, device)
    for b in range(7):  # poison what lies behind each row's last token in its last page
        n = int(case["seq_lens"][b])
        if n % 16:
            page = int(case["page_table"][b, n // 16])
            case["k_pool"][page, :, n % 16:] = float("inf")
            case["v_pool"][page, :, n % 16:] = float("nan")
    assert torch.equal(run_shared(case, device), clean)
    case = shared_case(10, [(3, 64)], [1, 9, 0], 4, 2)
    case["q"][:] = 1.0
    case["k_pool"][:] = -float("inf")
    assert torch.isnan(run_shared(case, device)).all()
    case["seq_lens"][1] = 0
    got = run_shared(case, device)
    assert bool((got[1] == 0).all()) and torch.isnan(got[[0, 2]]).all()


@pytest.mark.parametrize("rows,hq,hkv,prefix", [
    (3, 64, 64, 2048),     # 3 vectors of a KV head, about 12 blocks a piece: every wavefront meets both scores
    (40, 64, 16, 4096)])   # 160: a tile of 128 and one of 32
@pytest.mark.parametrize("low,high,times", [
    (2 ** 27 + 16, 2 ** 27 + 32, 1.0), (2 ** 26 + 8, 2 ** 26 + 16, 1.0), (2 ** 28 - 16, 2 ** 28, 1.0),
    (2 ** 24 + 2, 2 ** 24 + 10, 1.0), (-2 ** 27 - 32, -2 ** 27 - 16, 1.0),
    (89479112, 89479120, 1.5)])  # products 134218668 and ...680 round to ...672 and ...688
def test_shared_attention_scores_one_step_apart(device, rows, hq, hkv, prefix, low, high, times):
    """Scores so large that the next fp32 number is 2 to 16 further, every second 128 tokens the higher one.  The sums
    are exact here and the scale makes the exponents ``times`` the scores, rounded once, so a weight is 1 or 2 to their
    difference, and what is left are the roundings of the weights and the output and n sums in fp32."""
    scale = 0.6931471824645996 * times
    assert np.float32(scale) * np.float32(1.4426950408889634) == np.float32(times)
    case = shared_case(16, [(rows, prefix)], [(37 * b) % 50 + 1 for b in range(rows)], hq, hkv)
    parts = torch.tensor([2.0 ** 14, 2.0 ** 10, 2.0], dtype=torch.float64)
    case["q"].zero_()
    case["q"][:, :, :3] = parts.half()
    ref, tol = torch.zeros(case["q"].shape, dtype=torch.float64), torch.zeros(case["q"].shape, dtype=torch.float64)
    big = float(torch.tensor(high / 2 ** 14).half())
    for b in range(rows):
        n = int(case["seq_lens"][b])
        t = torch.arange(n)
        pages = case["page_table"][b].long()[t // 16]
        c = torch.where(t // 128 % 2 == 1, high, low).double()
        mid = ((c - big * 2 ** 14) / 2 ** 10).trunc()
        key = torch.zeros((n, hkv, 128), dtype=torch.float16)
        key[:, :, :3] = torch.stack([torch.full((n,), big, dtype=torch.float64), mid,
                                     (c - big * 2 ** 14 - mid * 2 ** 10) / 2], dim=1)[:, None].half()
        assert torch.equal(key[:, 0, :3].double() @ parts, c)
        case["k_pool"][pages, :, t % 16] = key
        v = case["v_pool"][pages, :, t % 16].double()
        s = (c * times).float().double()
        w = torch.exp2(s - s.max())
        l = w.sum()
        out, mass = ((w / l).view(-1, 1, 1).mul(x).sum(dim=0) for x in (v, v.abs()))
        off = mass * (2 * U16 + (n + 64) * U32) + v.abs().sum(dim=0) * 2.0 ** -25 / l + U16 * out.abs()
        ref[b], tol[b] = (x.repeat_interleave(hq // hkv, dim=0) for x in (out, off))
    got = run_shared(case, device, scale=scale)
    assert torch.isfinite(got).all()
    err = (got.cpu().double() - ref).abs()
    assert bool((err <= tol).all()), f"max excess {(err - tol).max():.3e}, max error {err.max():.3e}"


@pytest.mark.parametrize("slope", [0.002, 0.05, 0.17, 1.0, -0.05, -1.0])
@pytest.mark.parametrize("rows,hq,hkv", [(40, 8, 2), (3, 4, 1)])
def test_shared_attention_scores_that_rise_and_fall(device, slope, rows, hq, hkv):
    """Scores of slope * t: the running maximum is passed by little or much, once or in every block, and later pieces
    outweigh earlier ones (or weigh nothing)."""
    case = shared_case(14, [(rows, 640)], [(7 * b) % 300 for b in range(rows)], hq, hkv)
    sign = torch.randint(0, 2, (128,), generator=torch.Generator().manual_seed(0)) * 2.0 - 1.0
    case["q"] = (sign * (1 + torch.arange(rows * hq).view(rows, hq, 1) % 3 / 4)).half()
    for b in range(rows):
        t = torch.arange(int(case["seq_lens"][b]))
        pages = case["page_table"][b].long()[t // 16]
        case["k_pool"][pages, :, t % 16] = (sign * (slope * t / 128).view(-1, 1, 1)).half().expand(-1, hkv, -1)
    check_shared(case, run_shared(case, device, scale=1.0), 1.0)


def test_shared_attention_captured_and_on_a_stream(device):
    """Two graphs with workspaces of their own, replayed in turn with other lengths and prefixes between the replays,
    and a call on a stream of its own, all bit for bit the eager call's."""
    from cacheir_amd import kernels

    cases = [shared_case(11, [(20, 512), (3, 64)], list(range(1, 24)), 28, 4),
             shared_case(12, [(5, 96)], [100, 1, 2, 3, 200], 32, 8)]
    devs = [{k: v.to(device) for k, v in c.items()} for c in cases]
    outs = [torch.empty_like(d["q"]) for d in devs]
    graphs = []
    for d, o in zip(devs, outs):
        kernels.paged_decode_attention_shared(**d, out=o)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kernels.paged_decode_attention_shared(**d, out=o)
        graphs.append(g)
    for step in range(4):
        for d in devs:
            d["seq_lens"].sub_(step % 2)
            if step == 2:
                d["prefix_lens"].div_(2, rounding_mode="floor")
        for g in graphs:
            g.replay()
        got = [o.clone() for o in outs]
        for d, o in zip(devs, got):
            assert torch.equal(o, kernels.paged_decode_attention_shared(**d))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = kernels.paged_decode_attention_shared(**devs[0])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, got[0])


def test_shared_attention_refusals(device):
    case = shared_case(13, [(3, 96)], [1, 2, 3], 8, 2)
    with pytest.raises(TypeError, match="group_rows must be int32"):
        run_shared(case | {"group_rows": case["group_rows"].long()}, device)
    with pytest.raises(ValueError, match="group_rows must be"):
        run_shared(case | {"group_rows": case["group_rows"][:1].contiguous()}, device)
    with pytest.raises(TypeError, match="share a dtype"):
        run_shared(case | {"q": case["q"].float()}, device)
    with pytest.raises(RuntimeError, match="workspace too small"):
        run_shared(case, device, workspace=torch.empty(16, dtype=torch.uint8, device=device))
    with pytest.raises(ValueError, match="other pages"):
        t = case["page_table"].clone()
        t[1, 0] = t[1, 1]
        run_shared(case | {"page_table": t}, device, check_tables=True)
    with pytest.raises(ValueError, match="ascend"):
        run_shared(case | {"group_rows": torch.tensor([3, 0], dtype=torch.int32)}, device, check_tables=True)
    with pytest.raises(ValueError, match="on the GPU"):
        run_shared(case, "cpu")


# ---------------------------------------------------------------- page tables --
def tables_ref(table, lens, new, free, head, psize, max_tokens):
    """The loop over rows and tokens."""
    table, lens = table.clone(), lens.tolist()
    positions, slots, offsets, granted = [0] * max_tokens, [-1] * max_tokens, [0], []
    short = False
    for b, n in enumerate(new.tolist()):
        n = max(n, 0)
        at = offsets[-1]
        offsets.append(min(at + n, 2 ** 30))
        have, want = -(-lens[b] // psize), -(-(lens[b] + n) // psize)
        ok = want <= table.shape[1] and at + n <= max_tokens
        if ok and want > have:
            short = short or head + want - have > len(free)
            ok = not short
        if ok:
            for i in range(have, want):
                table[b, i] = free[head]
                head += 1
        for j in range(min(n, max_tokens - at)):
            p = lens[b] + j
            positions[at + j] = p
            if ok:
                slots[at + j] = int(table[b, p // psize]) * psize + p % psize
        granted.append(n if ok else 0)
        lens[b] += granted[-1]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    return [table, i32(lens), i32([head]), i32(offsets), i32(positions), torch.tensor(slots, dtype=torch.int64),
            i32(granted)]


def tables_case(seed, lens, new, psize=16, width=None, spare=4, taken=2):
    rng = np.random.default_rng(seed)
    have = [-(-n // psize) for n in lens]
    need = sum(max(0, -(-(n + max(a, 0)) // psize) - h) for n, a, h in zip(lens, new, have) if a < 10 ** 6)
    width = width or max([1] + [-(-(n + max(a, 0)) // psize) for n, a in zip(lens, new)])
    perm = rng.permutation(sum(have) + taken + need + max(spare, 0)).astype(np.int32)
    table = np.full((len(lens), width), 77777, dtype=np.int32)
    at = 0
    for b, h in enumerate(have):
        table[b, : min(h, width)] = perm[at: at + min(h, width)]
        at += h
    free = perm[sum(have): len(perm) + min(spare, 0)]
    t = lambda a: torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype=np.int32)))
    return dict(page_table=t(table), seq_lens=t(lens), new_tokens=t(new), free_slots=t(free), free_head=t([taken]))


def check_tables(case, device, psize, max_tokens):
    from cacheir_amd import kernels

    dev = {k: v.to(device) for k, v in case.items()}
    r = kernels.extend_page_tables(**dev, page_size=psize, max_tokens=max_tokens)
    got = [dev["page_table"], r.seq_lens, r.free_head, r.offsets, r.positions, r.slot_map, r.granted]
    want = tables_ref(case["page_table"], case["seq_lens"], case["new_tokens"], case["free_slots"].tolist(),
                      int(case["free_head"]), psize, max_tokens)
    for name, a, b in zip(("table", "lens", "head", "offsets", "positions", "slots", "granted"), got, want):
        assert torch.equal(a.cpu(), b), name
    assert torch.equal(dev["seq_lens"].cpu(), case["seq_lens"]) and torch.equal(dev["free_head"].cpu(), case["free_head"])


@pytest.mark.parametrize("lens,new,psize,width,spare,slack", [
    ([0], [1], 16, None, 4, 0),
    ([15, 16, 17, 31, 0], [1, 1, 1, 2, 0], 16, None, 4, 3),
    ([5, 0, 100], [0, 0, 0], 16, None, 0, 5),                 # nothing new
    ([5, 3], [-4, 2], 4, None, 4, 1),                         # a negative count is none
    ([0, 7, 64, 3], [3000, 1, 1, 500], 16, None, 4, 0),       # prompts: several workgroups
    ([30, 40, 50, 15, 3], [40, 40, 1, 1, 90], 16, None, -4, 0),  # the free slots run out
    ([30, 0, 16], [40, 500, 1], 16, 5, 4, 0),                 # a row too long for its table
    ([3, 4, 5], [10, 10, 10], 16, None, 4, -11),              # the map ends inside a row
    ([3, 9], [7, 7], 1, None, 2, 0),
    ([3, 9], [7, 2 ** 31 - 5], 16, 9, 2, 30 - 2 ** 31),       # a count no 32-bit sum or table holds
])
def test_page_tables(device, lens, new, psize, width, spare, slack):
    case = tables_case(len(lens), lens, new, psize, width, spare)
    check_tables(case, device, psize, sum(max(n, 0) for n in new) + slack)


@pytest.mark.parametrize("seed", range(6))
def test_page_tables_random(device, seed):
    rng = np.random.default_rng(seed)
    batch = int(rng.choice([1, 100, 256, 257, 700]))
    lens, new = rng.integers(0, 300, batch), rng.integers(0, int(rng.choice([2, 60])), batch)
    psize = int(rng.choice([16, 16, 5]))
    case = tables_case(seed, lens.tolist(), new.tolist(), psize, None, int(rng.choice([4, -3, -200])))
    check_tables(case, device, psize, max(0, int(new.sum()) + int(rng.integers(-3, 5))))


def test_page_tables_without_rows_or_tokens(device):
    from cacheir_amd import kernels

    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=device)
    r = kernels.extend_page_tables(z(0, 4), z(0), z(0), z(3), z(1) + 1, page_size=16, max_tokens=5)
    assert r.slot_map.tolist() == [-1] * 5 and r.positions.tolist() == [0] * 5
    assert r.offsets.tolist() == [0] and r.free_head.tolist() == [1]
    r = kernels.extend_page_tables(z(2, 4), z(2) + 3, z(2), z(0), z(1), page_size=16, max_tokens=0)
    assert r.seq_lens.tolist() == [3, 3] and r.offsets.tolist() == [0, 0, 0]


@pytest.mark.parametrize("step", [1, 700])
def test_page_tables_advance_in_place_under_a_graph(device, step):
    """A captured step whose lengths and head are updated in place, replayed: the states of one eager step after another
    (at 700 tokens a row the slot map takes several workgroups)."""
    from cacheir_amd import kernels

    lens, psize, rounds = [0, 15, 16, 200], 16, 4
    case = tables_case(3, lens, [step * rounds + 1] * 4, psize, None, 4)
    case["new_tokens"][:] = step
    dev = {k: v.to(device) for k, v in case.items()}
    out = kernels.StepTables.empty(4, 4 * step + 1, device)._replace(seq_lens=dev["seq_lens"], free_head=dev["free_head"])
    state = {k: v.clone() for k, v in dev.items()}
    call = lambda: kernels.extend_page_tables(**dev, page_size=psize, max_tokens=4 * step + 1, out=out)
    call()
    for k, v in state.items():
        dev[k].copy_(v)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    table, lens, head = case["page_table"], case["seq_lens"], int(case["free_head"])
    for _ in range(rounds):
        want = tables_ref(table, lens, case["new_tokens"], case["free_slots"].tolist(), head, psize, 4 * step + 1)
        g.replay()
        torch.cuda.synchronize()
        got = [dev["page_table"], out.seq_lens, out.free_head, out.offsets, out.positions, out.slot_map, out.granted]
        for a, b in zip(got, want):
            assert torch.equal(a.cpu(), b)
        table, lens, head = want[0], want[1], int(want[2])


def test_page_tables_refusals(device):
    from cacheir_amd import kernels

    case = {k: v.to(device) for k, v in tables_case(1, [3, 4], [1, 1]).items()}
    call = lambda page_size=16, max_tokens=4, out=None, **kw: kernels.extend_page_tables(
        **(case | kw), page_size=page_size, max_tokens=max_tokens, out=out)
    with pytest.raises(ValueError, match="page_size must be positive"):
        call(page_size=0)
    with pytest.raises(TypeError, match="seq_lens must be int32"):
        call(seq_lens=case["seq_lens"].long())
    with pytest.raises(ValueError, match="new_tokens must be"):
        call(new_tokens=case["new_tokens"][:1].contiguous())
    with pytest.raises(ValueError, match="contiguous"):
        call(page_table=case["page_table"].repeat(1, 2)[:, ::2])
    with pytest.raises(ValueError, match="out.positions"):
        call(out=kernels.StepTables.empty(2, 3, device))


# ------------------------------------------------------------- rotary append --
def rope64(x, positions, freq, factor, layout):
    """(turned, tolerance before the rounding to the output type)."""
    rot = 2 * freq.numel()
    y, tol = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    a = positions.double()[:, None] * freq[None]
    c, s = (torch.cos(a) * factor)[:, None], (torch.sin(a) * factor)[:, None]
    i = torch.arange(rot // 2)
    re, im = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + rot // 2)
    xr, xi = x.double()[..., re], x.double()[..., im]
    y[..., re], y[..., im] = xr * c - xi * s, xr * s + xi * c
    tol[..., re] = tol[..., im] = 10 * U32 * factor * (xr.abs() + xi.abs())
    return y, tol


@pytest.mark.parametrize("tokens,hq,hkv,d,rot,layout,dtype,kvdt,psize", [
    (1, 4, 2, 64, 64, "interleaved", torch.float32, torch.float32, 16),
    (33, 32, 8, 128, 128, "interleaved", torch.float16, torch.float16, 16),
    (70, 28, 4, 128, 64, "half", torch.float16, torch.float16, 16),
    (5, 8, 8, 80, 40, "half", torch.float16, torch.float16, 5),
    (7, 3, 1, 96, 24, "interleaved", torch.float16, torch.float32, 16),
    (9, 2, 2, 128, 32, "half", torch.float32, torch.float16, 32),
    (6, 5, 1, 34, 10, "half", torch.float32, torch.float32, 7),
    (4, 3, 3, 34, 34, "interleaved", torch.float16, torch.float16, 16),
    (3, 2, 1, 256, 256, "half", torch.float16, torch.float16, 16),
    (3, 2, 1, 2, 2, "half", torch.float32, torch.float32, 16),
    (5, 4, 2, 64, 0, "half", torch.float16, torch.float16, 16),
])
def test_rope_append(device, tokens, hq, hkv, d, rot, layout, dtype, kvdt, psize):
    """Views of one projection, positions up to 2^20, a scaled table, some padding tokens, untouched slots."""
    from cacheir_amd import kernels

    g = torch.Generator().manual_seed(tokens * d + rot)
    qkv = torch.randn((tokens, (hq + 2 * hkv) * d + 3 * (d % 4 == 0) * 8), generator=g).to(dtype)
    cut = lambda t: [x.unflatten(1, (-1, d)) for x in t[:, : (hq + 2 * hkv) * d].split([hq * d, hkv * d, hkv * d], dim=1)]
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g).int()
    pages = -(-tokens // psize) + 2
    slots = torch.randperm(pages * psize, generator=g)[:tokens]
    if tokens > 4:
        slots[1], slots[3], pos[1] = -1, pages * psize, -7
    freq = kernels.rope_frequencies(rot, 500000.0, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
                                                    "high_freq_factor": 4.0, "original_max_position_embeddings": 8192},
                                    device)
    factor = 1.25
    pools = [torch.randn((pages, hkv, psize, d), generator=g).to(kvdt) for _ in range(2)]
    kp, vp = (p.to(device) for p in pools)
    q, k, v = cut(qkv)
    dq, dk, dv = cut(qkv.to(device))
    out = torch.full((tokens, hq, d), 9.0, dtype=dtype, device=device)
    got = kernels.rope_append(dq, dk, dv, pos.to(device), slots.to(device), freq, kp, vp, layout=layout, factor=factor,
                              out=out)
    assert got.data_ptr() == out.data_ptr()
    live = (slots >= 0) & (slots < pages * psize)
    for x, res, rd in ((q, got.cpu(), dtype), (k, None, kvdt)):
        ref, tol = rope64(x, pos, freq.cpu(), factor, layout)
        if res is None:
            want = pools[0].double().transpose(1, 2).reshape(pages * psize, hkv, d)
            want[slots[live]] = ref[live]
            wtol = torch.zeros_like(want)
            wtol[slots[live]] = tol[live] + (U16 if rd == torch.float16 else U32) * ref[live].abs()
            have = kp.cpu().double().transpose(1, 2).reshape(pages * psize, hkv, d)
            assert bool(((have - want).abs() <= wtol).all())
        else:
            assert bool((res[~live] == 9.0).all())
            err, wtol = (res.double() - ref).abs(), tol + (U16 if rd == torch.float16 else U32) * ref.abs()
            assert bool((err[live] <= wtol[live]).all()), (err - wtol)[live].max()
    want = pools[1].clone().transpose(1, 2).reshape(pages * psize, hkv, d)
    want[slots[live]] = v[live].to(kvdt)
    assert torch.equal(vp.cpu().transpose(1, 2).reshape(pages * psize, hkv, d), want)
    # in place of q, and without a table entry: the same bits
    again = kernels.rope_append(dq, dk, dv, pos.to(device), slots.to(device), freq, kp, vp, layout=layout, factor=factor,
                                out=dq)
    assert torch.equal(again[live.to(device)], got[live.to(device)])


@pytest.mark.parametrize("tokens,hq,hkv,d,rot,layout,dtype,kvdt", [
    (5, 8, 8, 80, 20, "half", torch.float16, torch.float16),         # 10 pairs: no whole vectors of 4 or 8
    (9, 8, 8, 80, 20, "interleaved", torch.float16, torch.float32),
    (6, 4, 2, 128, 36, "half", torch.float32, torch.float16),
    (7, 16, 8, 96, 24, "half", torch.float16, torch.float16),        # vectors of 4 where the pools would take 8
    (130, 3, 1, 80, 78, "half", torch.float16, torch.float16),
])
def test_rope_append_of_parts_that_are_no_whole_vectors(device, tokens, hq, hkv, d, rot, layout, dtype, kvdt):
    test_rope_append(device, tokens, hq, hkv, d, rot, layout, dtype, kvdt, 16)


def test_rope_append_matches_the_step_epilogue(device):
    """Interleaved, whole head, small positions: the K and V pages of ``epilogue_qkv_rope_append`` within the rounding of
    its fp32 angle."""
    from cacheir_amd import kernels
    from cacheir_amd.runtime import rope_inv_freq

    rows, hq, hkv, d, P = 9, 8, 2, 128, 16
    part = torch.randn((1, rows, (hq + 2 * hkv) * d), device=device).half().float()
    pos = torch.arange(rows, dtype=torch.int32, device=device) * 3
    pt = torch.arange(rows * 2, dtype=torch.int32, device=device).view(rows, 2)
    pools = [torch.zeros((rows * 2, hkv, P, d), dtype=torch.float16, device=device) for _ in range(4)]
    q_old = torch.empty((rows, hq * d), dtype=torch.float16, device=device)
    inv = torch.from_numpy(rope_inv_freq(d, 10000.0)).to(device)
    kernels.epilogue_qkv_rope_append(part, inv, pos, pt, q_old, pools[0], pools[1], batch=rows, q_len=1, num_heads=hq,
                                     num_kv_heads=hkv, head_dim=d)
    q, k, v = (x.unflatten(1, (-1, d)) for x in part[0].half().split([hq * d, hkv * d, hkv * d], dim=1))
    slots = (pt[torch.arange(rows, device=device), (pos // P).long()].long() * P + pos % P)
    q_new = kernels.rope_append(q, k, v, pos, slots, inv.double(), pools[2], pools[3])
    assert torch.equal(pools[1], pools[3])
    # 5: |a| + |b| of N(0, 1) values here; the angles differ by their fp32 rounding, 24 * 3 * u32, then two roundings
    assert (q_new.view(rows, -1).float() - q_old.float()).abs().max() <= 10 * 2 * 72 * U32 + 2 * U16 * 7
    assert (pools[0].float() - pools[2].float()).abs().max() <= 10 * 2 * 72 * U32 + 2 * U16 * 7


def test_rope_append_to_the_halves_of_one_allocation(device):
    """K and V pools one behind the other in memory, as a stacked cache holds them; one tensor as both is refused."""
    from cacheir_amd import kernels

    x = torch.randn((9, 8, 64), device=device).half()
    pos, slots = (torch.arange(9, device=device, dtype=t) for t in (torch.int32, torch.int64))
    both, kp, vp = (torch.zeros((*n, 2, 2, 16, 64), dtype=torch.float16, device=device) for n in ((2,), (), ()))
    freq = kernels.rope_frequencies(64, 1e4, None, device)
    args = x[:, :4], x[:, 4:6], x[:, 6:], pos, slots, freq
    assert torch.equal(kernels.rope_append(*args, both[0], both[1]), kernels.rope_append(*args, kp, vp))
    assert torch.equal(both[0], kp) and torch.equal(both[1], vp)
    with pytest.raises(RuntimeError, match="k_pool and v_pool overlap"):
        kernels.rope_append(*args, kp, kp)


def test_rope_frequencies_by_the_formula():
    from cacheir_amd import kernels

    f = kernels.rope_frequencies(8, 10000.0, None, "cpu")
    assert torch.equal(f, torch.tensor([10000.0 ** (-i / 4) for i in range(4)], dtype=torch.float64))
    assert torch.equal(kernels.rope_frequencies(8, 10000.0, {"type": "linear", "factor": 4}, "cpu"), f / 4)
    s = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
             original_max_position_embeddings=8192)
    got, plain = kernels.rope_frequencies(128, 500000.0, s, "cpu"), kernels.rope_frequencies(128, 500000.0, None, "cpu")
    for a, b in zip(got.tolist(), plain.tolist()):
        turns = 8192 * b / (2 * math.pi)
        keep = 1.0 if turns > 4 else 0.0 if turns < 1 else (turns - 1) / 3
        assert abs(a - (keep * b + (1 - keep) * b / 8)) <= 1e-15 * b
    with pytest.raises(ValueError, match="unsupported rope scaling"):
        kernels.rope_frequencies(8, 1e4, {"rope_type": "other"}, "cpu")


def test_rope_append_refusals(device):
    from cacheir_amd import kernels

    z = lambda *s, dtype=torch.float16: torch.zeros(s, dtype=dtype, device=device)
    base = dict(q=z(2, 4, 64), k=z(2, 2, 64), v=z(2, 2, 64), positions=z(2, dtype=torch.int32),
                slot_map=z(2, dtype=torch.int64), inv_freq=z(32, dtype=torch.float64), k_pool=z(3, 2, 16, 64),
                v_pool=z(3, 2, 16, 64))
    for kw, exc, match in [(dict(k=z(2, 2, 64, dtype=torch.float32)), TypeError, "share a dtype"),
                           (dict(k=z(2, 3, 64)), ValueError, "k and v must be"),
                           (dict(q=z(2, 4, 65)[:, :, ::2]), ValueError, "contiguous heads"),
                           (dict(inv_freq=z(33, dtype=torch.float64)), ValueError, "turns 66 dims"),
                           (dict(inv_freq=z(32, dtype=torch.float32)), TypeError, "inv_freq must be float64"),
                           (dict(slot_map=z(2, dtype=torch.int32)), TypeError, "slot_map must be int64"),
                           (dict(v_pool=z(4, 2, 16, 64)), ValueError, "v_pool must be"),
                           (dict(layout="other"), ValueError, "layout must be"),
                           (dict(out=z(2, 4, 32)), ValueError, "out must be like q")]:
        with pytest.raises(exc, match=match):
            kernels.rope_append(**(base | kw))
    with pytest.raises(RuntimeError, match="head_dim 300"):
        kernels.rope_append(z(2, 4, 300), z(2, 2, 300), z(2, 2, 300), base["positions"], base["slot_map"],
                            base["inv_freq"], z(3, 2, 16, 300), z(3, 2, 16, 300))


# --------------------------------------------------------- log probabilities --
def check_logprobs(logits, ids, k, r, which=None):
    """``logits`` on the CPU (any dtype), rows without NaN or +inf; row i of the results is of logits row ``which[i]``."""
    rows, vocab = logits.shape
    which = torch.arange(rows) if which is None else which
    x = logits.double()
    lp = torch.log_softmax(x, dim=1)
    p = lp.exp()
    h = -(torch.where(p > 0, p * lp, 0.0)).sum(dim=1)
    sums = (vocab / 256 + 100 + 8) * U32
    m = x.max(dim=1, keepdim=True).values
    near = lambda got, want, tol: bool((((got.cpu().double() - want).abs() <= tol) | (got.cpu().double() == want)).all())
    order = np.argsort(-x.numpy(), axis=1, kind="stable")[:, :k]
    order = torch.from_numpy(np.ascontiguousarray(order))
    assert torch.equal(r.top_ids.cpu(), order[which])
    best, away = lp.gather(1, order), (x.gather(1, order) - m).abs()
    assert near(r.top_logprobs, best[which], (sums + U32 * (away + best.abs()))[which])
    assert near(r.entropy, h[which], (2 * sums * (1 + h) + 2 * U32 * h)[which])
    if ids is not None:
        inside = (ids >= 0) & (ids < vocab)
        at = ids.clamp(0, vocab - 1)
        want, d = lp[which, at], (x[which, at] - m[which, 0]).abs()
        got = r.logprobs.cpu()
        assert torch.isnan(got[~inside]).all()
        assert near(got[inside], want[inside], (sums + U32 * (d + want.abs()))[inside])


@pytest.mark.parametrize("rows,vocab,k,dtype,pad", [
    (1, 1, 0, torch.float32, 0), (1, 1, 1, torch.float16, 0), (3, 7, 7, torch.float32, 1), (2, 64, 64, torch.float16, 3),
    (5, 1000, 5, torch.float32, 0), (4, 1023, 20, torch.float16, 5), (1, 128256, 20, torch.float32, 0),
    (33, 16384, 64, torch.float32, 1), (600, 515, 3, torch.float16, 0), (2, 152064, 1, torch.float16, 8),
    (700, 8200, 2, torch.float32, 0),
])
def test_logprobs(device, rows, vocab, k, dtype, pad):
    from cacheir_amd import kernels

    g = torch.Generator().manual_seed(rows + vocab)
    wide = (torch.randn((rows, vocab + pad), generator=g) * 3).to(dtype)
    ids = torch.randint(-2, vocab + 2, (rows,), generator=g)
    dev = wide.to(device)
    r = kernels.token_logprobs(dev[:, :vocab], ids.to(device), k)
    assert r.top_ids.shape == (rows, k) and r.top_logprobs.shape == (rows, k)
    check_logprobs(wide[:, :vocab], ids, k, r)
    assert kernels.token_logprobs(dev[:, :vocab], None, 0).logprobs is None


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("vocab", [300, 20000])
def test_logprobs_ties_order_and_masks(device, dtype, vocab):
    """Equal values, ascending and descending rows, masks of -inf and of the type's lowest value, far offsets."""
    from cacheir_amd import kernels

    g = torch.Generator().manual_seed(vocab)
    low = torch.finfo(dtype).min
    ramp = torch.linspace(-8, 8, vocab)
    rows = [torch.zeros(vocab), ramp, ramp.flip(0), torch.randint(-3, 3, (vocab,), generator=g).float(),
            torch.randn(vocab, generator=g).masked_fill(torch.rand(vocab, generator=g) < 0.9, -math.inf),
            torch.randn(vocab, generator=g).masked_fill(torch.rand(vocab, generator=g) < 0.9, low),
            torch.full((vocab,), low), torch.randn(vocab, generator=g) - (60000 if dtype == torch.float16 else 1e6)]
    one = torch.full((vocab,), -math.inf)
    one[vocab // 2] = 5.0
    rows.append(one)
    x = torch.stack(rows).to(dtype)
    ids = torch.randint(0, vocab, (len(rows),), generator=g)
    check_logprobs(x, ids, 20, kernels.token_logprobs(x.to(device), ids.to(device), 20))


@pytest.mark.parametrize("rows,vocab,dtype", [
    (1100, 100, torch.float32), (1100, 100, torch.float16), (1027, 700, torch.float32), (1027, 1900, torch.float16),
    (1100, 3000, torch.float32), (1030, 8000, torch.float16),           # a wavefront per row, one group and several
    (520, 90001, torch.float32), (516, 180000, torch.float16), (513, 5000, torch.float32)])  # a workgroup per row
def test_logprobs_many_rows(device, rows, vocab, dtype):
    """Copies of a dozen rows (random, rising, equal, masked but for a few, one value repeated, NaN) under other ids."""
    from cacheir_amd import kernels

    g = torch.Generator().manual_seed(rows + vocab)
    few = torch.full((vocab,), -math.inf)
    few[torch.randint(0, vocab, (3,), generator=g)] = 1.5
    half = torch.randn(vocab, generator=g)
    half[vocab // 3:] = 2.0
    kinds = [torch.linspace(-8, 8, vocab), torch.zeros(vocab), few, half,
             torch.randn(vocab, generator=g).masked_fill(torch.rand(vocab, generator=g) < 0.99, torch.finfo(dtype).min)]
    kinds += [torch.randn(vocab, generator=g) * 4 for _ in range(6)]
    x = torch.stack(kinds).to(dtype)
    which = torch.arange(rows) % len(kinds)
    ids = torch.randint(0, vocab, (rows,), generator=g)
    r = kernels.token_logprobs(x.to(device)[which.to(device)].contiguous(), ids.to(device), 7)
    check_logprobs(x, ids, 7, r, which)
    bad = x.clone()
    bad[:, vocab // 2] = math.nan
    r = kernels.token_logprobs(bad.to(device)[which.to(device)].contiguous(), ids.to(device), 7)
    order = [vocab // 2] + [i for i in np.argsort(-x[5].float().numpy(), kind="stable")[:8].tolist() if i != vocab // 2]
    assert r.top_ids[5].tolist() == order[:7] and torch.isnan(r.entropy).all() and torch.isnan(r.logprobs).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_logprobs_of_a_likely_token_among_many_unlikely_ones(device, dtype):
    """1 + 150000 times 1e-8: added one by one to the 1, some 600 of a thread's terms (6e-6) would be lost.  A thread adds
    19 groups of 32 (38 of 16) sums to it and 12 joins follow, each off by 2^-24 at most; the rest is exact to 2e-10."""
    from cacheir_amd import kernels

    rows, vocab, low = 512, 150001, -18.40625
    x = torch.full((rows, vocab), low, dtype=dtype, device=device)
    ids = (torch.arange(rows, device=device) * 293) % vocab
    x[torch.arange(rows, device=device), ids] = 0.0
    got = kernels.token_logprobs(x, ids, 2)
    want = -np.log1p((vocab - 1) * np.exp(low))
    bound = (19 + 12 if dtype == torch.float16 else 38 + 12) * U32 + 2e-10
    assert float((got.logprobs.double() - want).abs().max()) <= bound
    assert torch.equal(got.top_ids[:, 0], ids) and torch.equal(got.top_logprobs[:, 0], got.logprobs)


def test_logprobs_rows_without_probabilities(device):
    """NaN, +inf, and -inf alone: NaN probabilities; the order stays (NaN first, then by value, then by index)."""
    from cacheir_amd import kernels

    for vocab in (500, 9000):
        x = torch.randn((4, vocab))
        x[0, [3, 77, vocab - 1]] = math.nan
        x[1, [9, 400]] = math.inf
        x[2] = -math.inf
        r = kernels.token_logprobs(x.to(device), torch.zeros(4, dtype=torch.int64, device=device), 4)
        assert torch.isnan(r.logprobs[:3]).all() and torch.isnan(r.entropy[:3]).all()
        assert torch.isnan(r.top_logprobs[:3]).all() and torch.isfinite(r.top_logprobs[3]).all()
        best = lambda row, skip: int(torch.where(torch.isfinite(x[row]), x[row], -1e30).argmax())
        assert r.top_ids[0].tolist() == [3, 77, vocab - 1, best(0, 0)]
        assert r.top_ids[1, :3].tolist() == [9, 400, best(1, 0)]
        assert r.top_ids[2].tolist() == [0, 1, 2, 3]


@pytest.mark.parametrize("rows,vocab,dtype", [
    (1031, 1029, torch.float32), (1031, 3001, torch.float32), (1031, 4095, torch.float32),   # a wavefront per row,
    (1031, 2051, torch.float16), (1031, 8189, torch.float16),                                # several groups each
    (517, 4999, torch.float32), (517, 20001, torch.float32), (517, 20003, torch.float16),    # a workgroup per row
    (26, 60001, torch.float32), (32, 140007, torch.float16)])                                # several workgroups per row
def test_logprobs_equal_values_by_index(device, rows, vocab, dtype):
    """Rows of equal values and plateaus of the largest value that begin in every wavefront's share (and none, a few or
    many values before the end), where the values behind the last whole vector are equal too: the lowest ids win.  Rows
    lie next to one another, so they begin and end at every place within 16 bytes."""
    from cacheir_amd import kernels

    n = 4 if dtype == torch.float32 else 8  # values of a vector; a wavefront's turn is 64 of them
    assert vocab % 2 == 1
    low = -torch.rand(vocab, generator=torch.Generator().manual_seed(vocab)) * 4 - 1
    starts = [0, 3, 64 * n, 128 * n, 192 * n, 192 * n + 5, 256 * n + 64 * n, vocab // 2, vocab - 70 * n, vocab - n - 2,
              vocab - 1] + [max(0, vocab - turns * 64 * n) for turns in (8, 9, 10, 11)]
    kinds = []
    for at in starts:
        row = low.clone()
        row[min(at, vocab - 1):] = 2.0
        kinds.append(row)
    few = torch.full((vocab,), -math.inf)  # fewer than top_k tokens left
    few[[vocab // 3, vocab - 1]] = 1.0
    kinds += [few, torch.full((vocab,), torch.finfo(dtype).min)]
    x = torch.stack(kinds).to(dtype)  # 17 kinds: each meets every alignment
    which = torch.arange(rows) % len(kinds)
    dev = x.to(device)[which.to(device)].contiguous()
    for k in (1, 2, 3, 5, 7):
        check_logprobs(x, None, k, kernels.token_logprobs(dev, None, k), which)


def test_logprobs_graph_stream_and_refusals(device):
    from cacheir_amd import kernels

    x = torch.randn((3, 20000), device=device)
    ids = torch.tensor([1, 2, 19999], device=device)
    kernels.token_logprobs(x, ids, 8)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = kernels.token_logprobs(x, ids, 8)
    for _ in range(3):
        x.normal_()
        g.replay()
        for a, b in zip(held, kernels.token_logprobs(x, ids, 8)):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r = kernels.token_logprobs(x, ids, 8)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(held, r))
    with pytest.raises(ValueError, match="top_k must be"):
        kernels.token_logprobs(x, ids, 65)
    with pytest.raises(ValueError, match="top_k must be"):
        kernels.token_logprobs(x[:, :5], ids, 6)
    with pytest.raises(TypeError, match="unsupported dtype"):
        kernels.token_logprobs(x.double(), ids)
    with pytest.raises(TypeError, match="ids must be int64"):
        kernels.token_logprobs(x, ids.int())
    with pytest.raises(ValueError, match="contiguous rows"):
        kernels.token_logprobs(x[:, ::2], ids)
    with pytest.raises(ValueError, match="overlap"):
        kernels.token_logprobs(x[:1].expand(3, -1), ids)
    with pytest.raises(RuntimeError, match="workspace too small"):
        kernels.token_logprobs(x, ids, 8, workspace=torch.empty(8, dtype=torch.uint8, device=device))


# ------------------------------------------------------------------------ far --
def test_pages_past_32_bit_offsets(device):
    """Pages whose elements lie past 2^32 in their pools: what is appended there and read from there has the bits of the
    same pages at the start of small pools.  Logits of rows that lie 2^32 elements
    apart likewise."""
    from cacheir_amd import kernels

    case = shared_case(15, [(3, 96), (1, 0)], [5, 40, 17, 33], 8, 2)
    near = {k: v.to(device) for k, v in case.items()}
    pages = case["k_pool"].shape[0]
    first = (1 << 32) // case["k_pool"][0].numel() - pages // 2  # the pages lie on both sides of 2^32
    far = dict(near, page_table=near["page_table"] + first)
    for name in ("k_pool", "v_pool"):
        far[name] = torch.empty((first + pages, *near[name].shape[1:]), dtype=torch.float16, device=device)
        far[name][first:] = near[name]
    assert far["k_pool"].numel() > 1 << 32
    g = torch.Generator().manual_seed(0)
    x = torch.randn((pages, 12, 128), generator=g).half().to(device)
    pos = torch.arange(pages, dtype=torch.int32, device=device) * 1000
    freq = kernels.rope_frequencies(128, 1e4, None, device)
    slot = torch.arange(pages, device=device) * 16 + 3  # one token in every page
    outs = [kernels.rope_append(x[:, :8], x[:, 8:10], x[:, 10:], pos, slot + at * 16, freq, c["k_pool"], c["v_pool"])
            for c, at in ((near, 0), (far, first))]
    assert torch.equal(*outs)
    for name in ("k_pool", "v_pool"):
        assert torch.equal(far[name][first:], near[name])
    assert torch.equal(kernels.paged_decode_attention_shared(**far), kernels.paged_decode_attention_shared(**near))

    rows = torch.as_strided(far["k_pool"].view(-1), (2, 1000), ((1 << 32) - 1000, 1))  # the second ends at 2^32
    rows.copy_(torch.randn((2, 1000), generator=g))
    ids = torch.tensor([5, 999], device=device)
    for a, b in zip(kernels.token_logprobs(rows, ids, 4), kernels.token_logprobs(rows.contiguous(), ids, 4)):
        assert torch.equal(a, b)


def test_sizes_past_32_bits_are_refused(device):
    """Sizes that a C int does not hold (ctypes would pass their low 32 bits: a vocabulary of 5 for 2^32 + 5, the first
    page for a table of 2^32 + 1)."""
    from cacheir_amd import kernels

    far = (1 << 32) + 5
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=device)
    for kw in (dict(page_size=far, max_tokens=4), dict(page_size=16, max_tokens=far)):
        with pytest.raises(ValueError, match="32 bits"):
            kernels.extend_page_tables(i32(2, 4), i32(2), i32(2), i32(8), i32(1), **kw)
    with pytest.raises(ValueError, match="32 bits"):
        kernels.token_logprobs(torch.empty((1, far), dtype=torch.float16, device=device), None, 3)
    q, pool = (torch.zeros(s, dtype=torch.float16, device=device) for s in ((1, 8, 128), (4, 2, 16, 128)))
    with pytest.raises(ValueError, match="32 bits"):
        kernels.paged_decode_attention_shared(q, pool, pool, torch.empty((1, far), dtype=torch.int32, device=device), i32(1),
                                              i32(2), i32(1))
    k, none = (torch.empty((n, far, 2), dtype=torch.float16, device=device) for n in (1, 0))
    with pytest.raises(ValueError, match="32 bits"):
        kernels.rope_append(torch.zeros((1, 1, 2), dtype=torch.float16, device=device), k, k, i32(1), i32(1).long(),
                            torch.zeros(1, dtype=torch.float64, device=device), none.unsqueeze(2), none.unsqueeze(2))


# ------------------------------------------------------------------- together --
def test_decode_steps_of_the_operators_together(device):
    """Samples of two prompts: pages and slots built on the GPU, rotary append, attention over the shared prefixes and
    the log probabilities of the chosen tokens, captured once and replayed for some steps, against the same steps in
    float64 over contiguous caches (fp16 K and V as stored).  Keys, values and logits are fixed functions of the step."""
    from cacheir_amd import kernels

    hq, hkv, d, P, steps, vocab = 8, 2, 128, 16, 20, 5000
    groups, prefixes = [3, 2], [64, 100]
    batch = sum(groups)
    g = torch.Generator().manual_seed(0)
    case = shared_case(1, list(zip(groups, prefixes)), [5, 40, 1, 17, 3], hq, hkv, P, extra=40)
    lens0 = case["seq_lens"].clone()
    width = case["page_table"].shape[1] + 4
    table0 = torch.zeros((batch, width), dtype=torch.int32)
    table0[:, : case["page_table"].shape[1]] = case["page_table"]
    used = set()
    for b in range(batch):
        used |= set(table0[b, : -(-int(lens0[b]) // P)].tolist())
    free = torch.tensor([s for s in range(case["k_pool"].shape[0]) if s not in used], dtype=torch.int32)
    freq = kernels.rope_frequencies(d // 2, 1e4, None, device)
    qkv = (torch.randn((steps, batch, (hq + 2 * hkv) * d), generator=g)).half()
    head_w = (torch.randn((vocab, hq * d), generator=g) / 8)

    # on the GPU: static buffers, one captured step
    dev = lambda t: t.to(device)
    table, lens, head, fs = dev(table0), dev(lens0), torch.zeros(1, dtype=torch.int32, device=device), dev(free)
    kp, vp, gr, pl = (dev(case[k]) for k in ("k_pool", "v_pool", "group_rows", "prefix_lens"))
    one, x, w = torch.ones(batch, dtype=torch.int32, device=device), dev(qkv[0]), dev(head_w)
    st = kernels.StepTables.empty(batch, batch, device)._replace(seq_lens=lens, free_head=head)
    ids = torch.zeros(batch, dtype=torch.int64, device=device)

    def step():
        kernels.extend_page_tables(table, lens, one, fs, head, page_size=P, max_tokens=batch, out=st)
        q, k, v = (t.unflatten(1, (-1, d)) for t in x.split([hq * d, hkv * d, hkv * d], dim=1))
        q = kernels.rope_append(q, k, v, st.positions, st.slot_map, freq, kp, vp, layout="half")
        o = kernels.paged_decode_attention_shared(q, kp, vp, table, lens, gr, pl)
        logits = kernels.gemm_f32_partial(kernels.cast(o.view(batch, -1), torch.float32), w)[0]
        return o, logits, kernels.token_logprobs(logits, ids, 3)

    keep = [t.clone() for t in (table, lens, head, kp, vp)]
    step()
    torch.cuda.synchronize()
    for t, k in zip((table, lens, head, kp, vp), keep):
        t.copy_(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, logits, r = step()

    # the same on the CPU
    caches = []
    for b in range(batch):
        t = torch.arange(int(lens0[b]))
        pages = table0[b].long()[t // P]
        caches.append([case["k_pool"][pages, :, t % P], case["v_pool"][pages, :, t % P]])
    for s in range(steps):
        x.copy_(qkv[s])
        ids.copy_(torch.arange(batch) * 7 + s)
        graph.replay()
        torch.cuda.synchronize()
        pos = lens0 + s
        q, k, v = (t.unflatten(1, (-1, d)) for t in qkv[s].split([hq * d, hkv * d, hkv * d], dim=1))
        (qr, qt), (kr, kt) = (rope64(t, pos, freq.cpu(), 1.0, "half") for t in (q, k))
        for b in range(batch):
            # the stored key, checked, then taken as it is (fp16), so that errors do not pile up over the steps
            p = int(pos[b])
            page, off = int(table[b, p // P]), p % P
            stored = kp[page, :, off].cpu()
            assert bool(((stored.double() - kr[b]).abs() <= kt[b] + U16 * kr[b].abs()).all())
            assert torch.equal(vp[page, :, off].cpu(), v[b])
            caches[b][0] = torch.cat([caches[b][0], stored[None]])
            caches[b][1] = torch.cat([caches[b][1], v[b][None]])
            kc, vc = (c.double() for c in caches[b])
            for h in range(hkv):
                heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                sc = qr[b, heads] @ kc[:, h].T * d ** -0.5
                # q is stored in fp16: a score off by (qt + U16 |q|) |k|, on top of the fp32 sums
                off_s = ((qt + U16 * qr.abs())[b, heads] + 260 * U32 * qr[b, heads].abs()) @ kc[:, h].abs().T * d ** -0.5
                e = torch.exp(sc - sc.max(dim=1, keepdim=True).values)
                l = e.sum(dim=1, keepdim=True)
                ref, mass = e / l @ vc[:, h], e / l @ vc[:, h].abs()
                off_s = off_s.max(dim=1, keepdim=True).values
                tol = mass * (2 * U16 + 2 * off_s) + vc[:, h].abs().sum(0) * 2.0 ** -25 / l + U16 * ref.abs()
                err = (o[b, heads].cpu().double() - ref).abs()
                assert bool((err <= tol).all()), (s, b, h, (err - tol).max())
        check_logprobs(logits.cpu(), ids.cpu(), 3, r)
    assert torch.equal(lens.cpu(), lens0 + steps)
