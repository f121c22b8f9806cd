"""Refusals of the entry points for drafted trees that the host decides (no GPU calls)."""
import pytest
import torch

from cacheir_amd import hip, kernels

pytestmark = pytest.mark.skipif(not hip.library_path().exists(), reason="libcacheir_hip.so not built")

F16, F32 = hip.CIR_F16, hip.CIR_F32


def refuses(name, match, *args):
    with pytest.raises(RuntimeError, match=match):
        hip.call(name, *args)


def test_draft_tree_refusals():
    def call(match, tokens=4, batch=2, words=1, p=None):
        refuses("cir_draft_tree", match, p, p, p, p, p, p, tokens, batch, words, None)

    call("bad sizes", tokens=-1)
    call("bad sizes", batch=-1)
    call("words must be", words=0)
    call("words must be", words=5)
    call(r"2\^24", batch=1 << 24)
    call("tokens of no row", batch=0)
    call("null pointer")
    hip.call("cir_draft_tree", *[None] * 6, 0, 2, 1, None)


def test_accept_refusals():
    p, q = torch.zeros(64), torch.zeros(64)

    def call(match, dt=F32, slots=4, total=0, tokens=4, batch=2, most=4, pages=4, layers=1, heads=1, d=4, page=4, x=None,
             pools=(None, None), free=(None, None)):
        refuses("cir_accept_drafts", match, x, x, x, x, x, x, x, x, x, x, x, *pools, dt, slots, free[0], total, free[1], tokens,
                batch, most, pages, layers, heads, d, page, None)

    for kw in (dict(tokens=-1), dict(batch=-1), dict(layers=-1), dict(slots=-1), dict(total=-1)):
        call("bad sizes", **kw)
    call("most must be", most=0)
    call("most must be", most=257)
    call("bad dtype", dt=5)
    for kw in (dict(heads=0), dict(heads=4097), dict(d=0), dict(d=4097), dict(page=0), dict(pages=0), dict(layers=4097)):
        call("must be positive", **kw)
    call(r"2\^31 pages", slots=1 << 31)
    call(r"2\^31 pages", batch=1 << 20)
    call("null pointer")
    x = p.data_ptr()
    call("null pools", x=x)
    call("go together", x=x, pools=(x, q.data_ptr()), free=(x, None))
    call("overlap", x=x, pools=(x, x + 16))
    call(r"2\^30 parts", x=x, pools=(x, x + (1 << 50)), layers=4096, heads=4096, d=4095)
    hip.call("cir_accept_drafts", *[None] * 13, F32, 4, None, 0, None, 0, 0, 4, 4, 1, 1, 4, 4, None)


def test_adjust_logits_refusals():
    x = torch.zeros(64).data_ptr()

    def call(match, ld=100, out=None, ld_out=100, dt=F32, offsets=None, history=None, lens=None, width=0, drafts=None,
             masks=None, words=1, ids=None, bias=None, listed=0, rows=2, batch=2, vocab=100, logits=None):
        refuses("cir_adjust_logits", match, logits, ld, out, ld_out, dt, offsets, history, lens, None, width, drafts, masks,
                words, None, None, None, ids, bias, listed, None, rows, batch, vocab, None)

    call("bad dtype", dt=3)
    for kw in (dict(rows=-1), dict(batch=-1), dict(vocab=0)):
        call("bad sizes", **kw)
    call(r"2\^24 rows", rows=1 << 24, offsets=x)
    call(r"2\^16 sequences", batch=1 << 16, offsets=x)
    call(r"2\^30 tokens", vocab=(1 << 30) + 1, ld=1 << 31, ld_out=1 << 31)
    call("offsets do not name", rows=3)
    call("rows overlap", ld=99)
    call("rows overlap", ld_out=99)
    call("history of more", width=(1 << 20) - 256)
    call("more than 2047", listed=2048)
    call("words must be", drafts=x, words=5)
    call("words must be", drafts=x, words=0)
    call("null pointer")
    y = x + 4096
    call("null pointer", logits=x, out=y, history=x, width=4)
    call("null pointer", logits=x, out=y, drafts=x, offsets=x)
    call("null pointer", logits=x, out=y, ids=x, listed=1)
    call("drafts need offsets", logits=x, out=y, drafts=x, masks=x)
    call("overlaps", logits=x, out=x, ld_out=101)
    call("overlaps", logits=x, out=x + 796)
    call("overlaps", logits=x + 796, out=x)
    hip.call("cir_adjust_logits", None, 100, None, 100, F32, *[None] * 4, 0, None, None, 1, *[None] * 5, 0, None, 0, 0, 100, None)


@pytest.mark.parametrize("match,kw", [
    ("bad dtype", dict(dt=9)), ("bad dtype", dict(wdt=9)), ("bad dtype", dict(kvdt=9)), ("bad layout", dict(layout=2)),
    ("head_dim 7", dict(d=7)), ("head_dim 258", dict(d=258)), ("rotary_dim 10", dict(rot=10)), ("bad sizes", dict(tokens=-1)),
    ("whole pages", dict(slots=17)), (r"2\^26", dict(tokens=(1 << 26) + 1)), ("null pointer", {}),
    ("heads of q_out overlap", dict(p=4096, o=(16, 4))), ("other strides", dict(p=4096, o=(8, 16))),
    ("overlap", dict(p=4096, out=1 << 20)), ("null pointer", dict(p=4096, out=1 << 20, v_pool=1 << 30, w=None))])
def test_norm_rope_refusals(match, kw):
    def go(tokens=2, heads=2, kv_heads=1, d=8, rot=8, layout=0, dt=F32, kvdt=F32, wdt=F32, page=4, slots=16, q=(16, 8),
           o=(16, 8), p=None, out=None, v_pool=None, w=None):
        hip.call("cir_norm_rope_append", p, *q, p, 8, 8, p, 8, 8, dt, w, w, wdt, 1e-6, p, p, p, 1.0, rot, layout, out or p,
                 *o, p, v_pool or p, kvdt, slots, tokens, heads, kv_heads, d, page, None)

    with pytest.raises(RuntimeError, match="norm_rope_append.*" + match):
        go(**kw)
    go(tokens=0)


@pytest.mark.parametrize("bad", [(0, 1, 8, 2, 128, 16, 4), (2, 0, 8, 2, 128, 16, 4), (2, 1, 7, 2, 128, 16, 4),
                                 (2, 1, 8, 0, 128, 16, 4), (2, 1, 8, 2, 257, 16, 4), (2, 1, 8, 2, 128, 0, 4),
                                 (2, 1, 8, 2, 128, 16, 0), (2, 1, 8, 2, 128, 1 << 16, 1 << 16), (1 << 24, 1, 8, 2, 128, 16, 4)])
def test_tree_attention_workspace_of_bad_sizes(bad):
    assert hip.size_call("cir_tree_attention_workspace_bytes", *bad, F16) == 0


def test_tree_attention_refusals():
    def call(match, tokens=4, batch=2, hq=8, hkv=2, d=128, page=16, pages=4, dt=F16, words=1, p=None):
        refuses("cir_paged_tree_attention", match, *[p] * 8, words, p, None, 0, tokens, batch, hq, hkv, d, page, pages, 1.0, dt,
                None)

    p = torch.zeros(64).data_ptr()
    call("tokens and batch", tokens=-1)
    call("tokens and batch", batch=-1)
    call("null pointer")
    call("multiple of num_kv_heads", hq=7, p=p)
    call("head_dim 257", d=257, p=p)
    call("32-bit", page=1 << 16, pages=1 << 16, p=p)
    call("kv_dtype", dt=7, p=p)
    call("words must be", words=5, p=p)
    call("words must be", words=0, p=p)
    call(r"2\^26", tokens=1 << 23, p=p)
    call(r"2\^16 KV heads", hq=1 << 16, hkv=1 << 16, tokens=1, p=p)
    call(r"2\^20 rows", batch=1 << 20, p=p)
    call("workspace too small", pages=1000, p=p)
    hip.call("cir_paged_tree_attention", *[None] * 8, 1, None, None, 0, 0, 2, 8, 2, 128, 16, 4, 1.0, F16, None)


def test_sizes_past_a_c_int_are_refused(monkeypatch):
    monkeypatch.setattr(kernels, "_fits", lambda *a: True)
    with pytest.raises(ValueError, match="32 bits"):
        kernels._int32(1, 1 << 31)
