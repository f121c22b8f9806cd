"""Sizes and refusals of the serving operators' entry points that the host decides (no GPU calls)."""
import math

import pytest
import torch

from cacheir_amd import hip, kernels

pytestmark = pytest.mark.skipif(not hip.library_path().exists(), reason="libcacheir_hip.so not built")

F16, F32 = hip.CIR_F16, hip.CIR_F32


def refuses(name, match, *args):
    with pytest.raises(RuntimeError, match=match):
        hip.call(name, *args)


@pytest.mark.parametrize("batch,groups,hq,hkv", [(1, 0, 8, 8), (3, 1, 28, 4), (128, 16, 32, 8), (2048, 256, 32, 1)])
def test_shared_attention_workspace(batch, groups, hq, hkv):
    """Room for both paths (the pools' addresses, which a size query does not see, decide between them): at least the
    plain decode's, and fp32 (m, l, O) of every row's own piece and of a 128-vector prefix tile per group."""
    size = hip.size_call("cir_shared_attention_workspace_bytes", batch, groups, hq, hkv, 128, 16, 64, F16)
    assert size >= hip.size_call("cir_paged_attention_workspace_bytes", batch, hq, 128, 1024)
    assert size >= 4 * 130 * (batch * hq + groups * hkv * 128)
    for plain in ((64, 16, F16), (128, 16, F32), (128, 8, F16)):  # sizes that read each row alone
        d, page, dt = plain
        assert (hip.size_call("cir_shared_attention_workspace_bytes", batch, groups, hq, hkv, d, page, 64, dt)
                == hip.size_call("cir_paged_attention_workspace_bytes", batch, hq, d, 64 * page))


@pytest.mark.parametrize("page,prefix", [(64, 32), (64, 33), (64, 63), (64, 100), (48, 47), (48, 95), (16, 1), (16, 96)])
def test_checked_tables_cover_the_page_in_which_a_prefix_ends(monkeypatch, page, prefix):
    """Every page that holds a token of the prefix is the same in all rows of a group: the kernel reads whole 32-token
    blocks of the prefix from the first row's pages, the part of a page among them."""
    monkeypatch.setattr(kernels, "_cuda", lambda *a, **k: None)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    q, pool = torch.zeros(5, 8, 128, dtype=torch.float16), torch.zeros(40, 2, page, 128, dtype=torch.float16)
    table = torch.arange(35, dtype=torch.int32).view(5, 7)
    last = (prefix - 1) // page
    table[1:4, : last + 1] = table[1, : last + 1]
    check = lambda t: kernels._check_shared(q, pool, pool, t, i32([prefix + 1] * 5), i32([1, 4, 5]), i32([prefix, 40]),
                                            True)
    check(table)
    for col in range(last + 1):
        other = table.clone()
        other[3, col] = 39
        with pytest.raises(ValueError, match="group 0: rows with other pages"):
            check(other)
    other = table.clone()
    other[3, last + 1] = 39  # behind the prefix
    check(other)


@pytest.mark.parametrize("bad", [(0, 1, 8, 2, 128, 16, 4), (2, -1, 8, 2, 128, 16, 4), (2, 1, 7, 2, 128, 16, 4),
                                 (2, 1, 8, 0, 128, 16, 4), (2, 1, 8, 2, 0, 16, 4), (2, 1, 8, 2, 128, 0, 4),
                                 (2, 1, 8, 2, 128, 16, 0), (2, 1, 8, 2, 128, 1 << 16, 1 << 16)])
def test_shared_attention_workspace_of_bad_sizes(bad):
    assert hip.size_call("cir_shared_attention_workspace_bytes", *bad, F16) == 0


def test_shared_attention_refusals():
    def call(match, groups=1, batch=2, hq=8, hkv=2, d=128, page=16, pages=4, dt=F16, p=None):
        refuses("cir_paged_decode_attention_shared", match, p, p, p, p, p, None, None, groups, p, None, 0, batch, hq, hkv,
                d, page, pages, 1.0, dt, None)

    p = torch.zeros(64).data_ptr()
    call("batch and groups", groups=-1)
    call("batch and groups", batch=-1)
    call("null pointer")
    call("null group_rows", p=p)
    call("multiple of num_kv_heads", groups=0, hq=7, p=p)
    call("head_dim 257", groups=0, d=257, p=p)
    call("32-bit", groups=0, page=1 << 16, pages=1 << 16, p=p)
    call("kv_dtype", groups=0, dt=7, p=p)
    call("workspace too small", groups=0, p=p)
    hip.call("cir_paged_decode_attention_shared", *[None] * 7, 0, None, None, 0, 0, 8, 2, 128, 16, 4, 1.0, F16, None)


def test_page_tables_refusals():
    def call(match, free_total=4, batch=2, pages=4, page=16, tokens=8, p=None):
        refuses("cir_extend_page_tables", match, p, p, p, p, free_total, p, p, p, p, p, p, p, batch, pages, page, tokens,
                None)

    call("bad sizes", batch=-1)
    call("bad sizes", tokens=-1)
    call("bad sizes", free_total=-1)
    call("must be positive", page=0)
    call("must be positive", pages=0)
    call(r"2\^30", tokens=1 << 30)
    call(r"2\^30", free_total=1 << 30)
    call("null pointer")
    call("null pointer", batch=0)


def rope(tokens=2, heads=2, kv_heads=1, d=8, rot=8, layout=0, dt=F32, kvdt=F32, page=4, slots=16, q=(16, 8), o=(16, 8),
         p=None, out=None):
    hip.call("cir_rope_append", p, *q, p, 8, 8, p, 8, 8, dt, p, p, p, 1.0, rot, layout, out or p, *o, p, p, kvdt, slots,
             tokens, heads, kv_heads, d, page, None)


@pytest.mark.parametrize("match,kw", [
    ("bad dtype", dict(dt=9)), ("bad dtype", dict(kvdt=9)), ("bad layout", dict(layout=2)), ("head_dim 7", dict(d=7)),
    ("head_dim 258", dict(d=258)), ("rotary_dim 10", dict(rot=10)), ("rotary_dim 3", dict(rot=3)),
    ("bad sizes", dict(tokens=-1)), ("bad sizes", dict(kv_heads=0)), ("bad sizes", dict(page=0)),
    ("bad sizes", dict(slots=-1)), (r"2\^26", dict(tokens=(1 << 26) + 1)), (r"2\^20", dict(heads=(1 << 20) + 1)),
    ("null pointer", {})])
def test_rope_refusals(match, kw):
    with pytest.raises(RuntimeError, match=match):
        rope(**kw)


def test_rope_refuses_outputs_that_overlap():
    """Tokens or heads of q_out on one another (an expanded tensor), and q in place as a view with other strides."""
    x, y = torch.zeros(64), torch.zeros(64)
    for o in ((0, 8), (16, 0), (16, 4), (7, 8)):
        with pytest.raises(RuntimeError, match="overlap"):
            rope(p=x.data_ptr(), out=y.data_ptr(), o=o)
    with pytest.raises(RuntimeError, match="other strides"):
        rope(p=x.data_ptr(), o=(8, 16))
    rope(tokens=0)


def test_rope_refuses_exactly_the_outputs_that_overlap():
    """Token and head stride together, against the heads' elements counted out.  (q_out is q here, at strides that q does
    not have, so no call reaches a launch.)"""
    x = torch.zeros(64)
    for tokens, heads, d in ((2, 4, 8), (4, 2, 8), (3, 3, 4), (5, 2, 2), (1, 4, 8), (4, 1, 8)):
        strides = [s for s in range(-5 * d - 3, 5 * d + 4)]
        for ts in strides[:: 1 if d < 8 else 3] + [8, 16, 24, 32, -8, -32]:
            for hs in strides[:: 1 if d < 8 else 5] + [8, 16, 24, 32, -8, -32]:
                first = {t * ts + h * hs for t in range(tokens) for h in range(heads)}
                at = {e + i for e in first for i in range(d)}
                apart = len(at) == tokens * heads * d
                with pytest.raises(RuntimeError, match="other strides" if apart else "overlap"):
                    rope(tokens=tokens, heads=heads, d=d, rot=d, p=x.data_ptr(), o=(ts, hs), q=(999, 999))


@pytest.mark.parametrize("o", [(2 ** 63 - 1, -2 ** 63), (-2 ** 63, 8), (2 ** 40 + 1, 2 ** 40), (2 ** 62, 2 ** 62)])
def test_rope_overlap_of_far_strides(o):
    x = torch.zeros(64)
    for tokens, heads in ((1 << 20, 3), (3, 1 << 20), (2, 2)):
        # 1: t = h = 1 of (2^63 - 1, -2^63); 1 - 2^20 + ... of neighbours; equal strides
        match = "other strides" if o == (-2 ** 63, 8) else "overlap"
        with pytest.raises(RuntimeError, match=match):
            rope(tokens=tokens, heads=heads, p=x.data_ptr(), o=o, q=(16, 9))


def test_rope_refuses_pools_that_overlap():
    """K and V of different threads in the same elements: one tensor as both pools, or one that begins inside the other."""
    pools = torch.zeros(600)

    def call(k, v, slots=16, kvdt=F32):
        a, p = pools.data_ptr(), torch.zeros(64).data_ptr()
        refuses("cir_rope_append", "k_pool and v_pool overlap", p, 16, 8, p, 8, 8, p, 8, 8, F32, p, p, p, 1.0, 8, 0, p, 16,
                8, a + k, a + v, kvdt, slots, 2, 2, 1, 8, 4, None)

    size = 16 * 8 * 4  # slots x head_dim floats
    for k, v in ((0, 0), (0, 4), (size - 4, 0), (0, size - 4)):
        call(k, v)
    call(0, size // 2 - 2, kvdt=F16)


def test_rope_refuses_a_part_of_a_page():
    """Slots are whole pages: head 1 of a slot in a page cut short would lie behind the pool.  (The pools are one here: the
    last check, so that no call reaches a launch.)"""
    x = torch.zeros(64)
    for slots, page in ((17, 16), (15, 16), (1, 2), (2 ** 40 + 1, 4)):
        with pytest.raises(RuntimeError, match="whole pages"):
            rope(p=x.data_ptr(), slots=slots, page=page)
    for slots, page in ((16, 16), (2 ** 40, 4), (7, 1)):
        with pytest.raises(RuntimeError, match="k_pool and v_pool overlap"):
            rope(p=x.data_ptr(), slots=slots, page=page)


@pytest.mark.parametrize("tokens", [(1 << 26) - 3, 1 << 26])
def test_rope_refuses_launches_of_2_32_threads(tokens):
    """Four tokens to a workgroup of 256: 2^26 - 4 are the most whose rounded-up grid stays below 2^32 threads."""
    p = torch.zeros(64).data_ptr()
    with pytest.raises(RuntimeError, match=r"2\^26 - 4 tokens"):
        rope(tokens=tokens, p=p)
    with pytest.raises(RuntimeError, match="k_pool and v_pool overlap"):
        rope(tokens=(1 << 26) - 4, p=p)


@pytest.mark.parametrize("batch,hq,hkv", [
    (601, 111662, 3602),            # 2^26 - 2 query vectors, 31 a KV head: the join's 2^24 workgroups of 256
    (1, 1 << 25, 1 << 25),          # as many KV heads: a workgroup each in the first launch
    (1, 1 << 24, 1 << 24), (2, 1 << 23, 1 << 23)])  # (its record loop steps by 256 grids: 2^31)
def test_shared_attention_sizes_past_a_launch_read_each_row_alone(batch, hq, hkv):
    size = hip.size_call("cir_shared_attention_workspace_bytes", batch, 1, hq, hkv, 128, 16, 1, F16)
    assert size == hip.size_call("cir_paged_attention_workspace_bytes", batch, hq, 128, 16)
    less = hip.size_call("cir_shared_attention_workspace_bytes", batch, 1, hq // hkv * 1000, 1000, 128, 16, 1, F16)
    assert less > hip.size_call("cir_paged_attention_workspace_bytes", batch, hq // hkv * 1000, 128, 16)


def test_logprobs_workspace():
    """Nothing where a row has a workgroup of its own; 12 bytes of sums and top_k keys of 8 per split elsewhere."""
    size = lambda *a: hip.size_call("cir_token_logprobs_workspace_bytes", *a)
    assert size(512, 128256, 20) == size(1, 1000, 5) == size(0, 1000, 5) == size(4, 0, 5) == size(4, 100, -1) == 0
    one = size(3, 128256, 0)
    assert one > 0 and one % (3 * 12) == 0
    assert size(3, 128256, 20) == one // 12 * (12 + 160)


def test_logprobs_refusals():
    def call(match, dt=F16, ld=100, rows=2, vocab=100, k=5, p=None, ids=None):
        refuses("cir_token_logprobs", match, p, dt, ld, ids, rows, vocab, k, None, p, p, p, None, 0, None)

    p = torch.zeros(64).data_ptr()
    call("bad dtype", dt=9)
    call("bad sizes", rows=-1)
    call("bad sizes", vocab=0, k=0)
    call("bad sizes", ld=99)
    call("top_k 65", k=65)
    call("top_k 6", vocab=5, k=6)
    call("top_k -1", k=-1)
    call("null pointer")
    call("null pointer", p=p, ids=p)
    call("alignment", p=p + 1)
    call("workspace too small", p=p, rows=3, vocab=128256, ld=128256)
    call("too many", p=p, rows=1 << 26, vocab=5, ld=5)  # 2^24 workgroups of 256 threads
    call("too many", p=p, rows=1 << 24, vocab=5000, ld=5000)
    hip.call("cir_token_logprobs", None, F16, 100, None, 0, 100, 5, *[None] * 5, 0, None)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("vocab", [5, 1000, 5000, 100000])
def test_logprobs_of_too_many_rows_never_reach_a_launch(dt, vocab):
    """Status 1 is the argument check's own; a launch without a GPU fails with another one."""
    p = torch.zeros(64).data_ptr()
    for rows in (1 << 24, (1 << 26) + 1, 2 ** 31 - 1):
        refuses("cir_token_logprobs", "status 1: .*too many", p, dt, vocab, None, rows, vocab, 5, None, p, p, p, None, 0,
                None)


def test_rope_frequencies_on_the_host():
    f = kernels.rope_frequencies(8, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and torch.equal(f, 10000.0 ** (-torch.arange(4, dtype=torch.float64) / 4))
    assert torch.equal(kernels.rope_frequencies(8, 10000.0, {"rope_type": "linear", "factor": 4}, "cpu"), f / 4)
    assert kernels.rope_frequencies(0, 10000.0, device="cpu").numel() == 0
    scaled = kernels.rope_frequencies(128, 500000.0, {
        "rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
        "original_max_position_embeddings": 8192}, "cpu")
    plain = kernels.rope_frequencies(128, 500000.0, device="cpu")
    turns = plain * 8192 / (2 * math.pi)
    assert torch.equal(scaled[turns > 4], plain[turns > 4]) and torch.equal(scaled[turns < 1], plain[turns < 1] / 8)
    mid = (turns > 1) & (turns < 4)
    assert bool(((scaled[mid] < plain[mid]) & (scaled[mid] > plain[mid] / 8)).all()) and bool(mid.any())
    for bad in (dict(rotary_dim=3, theta=10000.0), dict(rotary_dim=8, theta=0.0),
                dict(rotary_dim=8, theta=10000.0, scaling={"rope_type": "other"})):
        with pytest.raises(ValueError):
            kernels.rope_frequencies(**bad, device="cpu")


def test_the_wrappers_refuse_host_tensors():
    i32 = lambda *n: torch.zeros(n, dtype=torch.int32)
    q, pool = torch.zeros(2, 8, 128, dtype=torch.float16), torch.zeros(4, 2, 16, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="on the GPU"):
        kernels.paged_decode_attention_shared(q, pool, pool, i32(2, 4), i32(2), i32(2), i32(1))
    with pytest.raises(ValueError, match="on the GPU"):
        kernels.extend_page_tables(i32(2, 4), i32(2), i32(2), i32(8), i32(1), page_size=16, max_tokens=2)
    with pytest.raises(ValueError, match="on the GPU"):
        kernels.rope_append(q, q[:, :2], q[:, :2], i32(2), i32(2).long(), torch.zeros(64, dtype=torch.float64), pool, pool)
    with pytest.raises(ValueError, match="on the GPU"):
        kernels.token_logprobs(torch.zeros(2, 100), torch.zeros(2, dtype=torch.int64))
