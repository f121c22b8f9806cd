"""Torch-tensor wrappers over the C ABI, with host-side shape/dtype/bounds checks.

Every wrapper checks on the host that operand shapes, dtypes, devices and
contiguity match what the kernel and its grid assume before anything is launched;
violations raise ``ValueError``/``TypeError`` (mirroring the reference runtime's
error types, ``cacheir/runtime/cuda.py:551-561``).  Page tables can additionally be
range-checked against the pool (``check_tables=True``; costs a device sync).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import NamedTuple

import torch

from cacheir_amd import hip
from cacheir_amd.hip import CIR_F16, CIR_F32, CIR_Q4_0, CIR_Q8_0

QK = 32
BLOCK_BYTES = {CIR_Q4_0: 18, CIR_Q8_0: 34}
FMT_NAMES = {"q4_0": CIR_Q4_0, "q8_0": CIR_Q8_0}


def _req(cond: bool, msg: str, exc=ValueError) -> None:
    if not cond:
        raise exc(msg)


def _cuda(t: torch.Tensor, name: str, rows_only: bool = False) -> None:
    """GPU tensor check; ``rows_only`` accepts a 2-D view whose rows are contiguous (any row stride)."""
    _req(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor", TypeError)
    _req(t.is_cuda, f"{name} must be on the GPU")
    if rows_only:
        _req(t.dim() == 2 and t.stride(1) == 1, f"{name} rows must be contiguous")
    else:
        _req(t.is_contiguous(), f"{name} must be contiguous")


def _call_on(dev: int, name: str, *args) -> None:
    """Launch on GPU ``dev``, on its current stream (it need not be the current GPU)."""
    if dev == torch._C._cuda_getDevice():
        hip.call(name, *args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            hip.call(name, *args, torch._C._cuda_getCurrentRawStream(dev))


def _fits(t, dev: int, dtype: torch.dtype, shape: tuple) -> bool:
    """A contiguous tensor of this type and shape on GPU ``dev``: the test of ``_tensors`` without its messages.  The
    wrappers of small launches ask this first (0.4 us a tensor against 1.5: page tables of 128 rows, 4.3 us of the GPU, took
    32 us of the host, now 12.5) and look for what is wrong only if something is."""
    return t.get_device() == dev and t.dtype is dtype and t.shape == shape and t.is_contiguous()


def _int32(*sizes: int) -> None:
    """Sizes that go to the library as C ints (ctypes passes the low 32 bits of larger ones)."""
    if max(sizes) >= 1 << 31:
        _req(False, f"sizes {sizes} do not fit 32 bits")


def _tensors(device: torch.device, **named: tuple) -> None:
    """Each of ``name=(tensor, dtype, shape)``: contiguous, on ``device``, of that dtype and shape."""
    for name, (t, dtype, shape) in named.items():
        _cuda(t, name)
        _req(t.device == device, f"{name} must be on {device}")
        _req(t.dtype == dtype, f"{name} must be {str(dtype).removeprefix('torch.')}", TypeError)
        _req(tuple(t.shape) == tuple(shape), f"{name} must be {list(shape)}, got {list(t.shape)}")


# ------------------------------------------------------------------ attention --
def attention_workspace(rows: int, num_heads: int, head_dim: int, max_context: int, device) -> torch.Tensor:
    n = hip.size_call("cir_paged_attention_workspace_bytes", rows, num_heads, head_dim, max_context)
    # holds split partials O and (max, sum), each written before it is read: no clearing needed
    return torch.empty(max(n, 4), dtype=torch.uint8, device=device)


def _check_pool(q, k_pool, v_pool, page_table, seq_lens, num_heads, check_tables):
    for t, n in ((q, "q"), (k_pool, "k_pool"), (v_pool, "v_pool"), (page_table, "page_table"), (seq_lens, "seq_lens")):
        _cuda(t, n)
    _req(k_pool.dtype == v_pool.dtype == q.dtype, "q, k_pool and v_pool must share a dtype", TypeError)
    _req(k_pool.dim() == 4 and v_pool.shape == k_pool.shape, "pools must be [slots, kv_heads, page_size, head_dim]")
    _req(page_table.dtype == torch.int32 and seq_lens.dtype == torch.int32, "page_table/seq_lens must be int32", TypeError)
    slots, kvh, psize, hd = k_pool.shape
    _req(num_heads % kvh == 0, f"num_heads {num_heads} must be a multiple of kv heads {kvh}")
    if check_tables and page_table.numel():
        _req(int(page_table.min()) >= 0 and int(page_table.max()) < slots, "page_table has slots outside the pool")
        _req(int(seq_lens.max()) <= page_table.shape[1] * psize, "seq_lens exceed the page table capacity")
    return slots, kvh, psize, hd


def paged_decode_attention(q, k_pool, v_pool, page_table, seq_lens, *, scale: float | None = None,
                           out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                           check_tables: bool = False) -> torch.Tensor:
    """q ``[B, Hq, D]`` -> out ``[B, Hq, D]`` over the paged context (decode, one query per sequence)."""
    _req(q.dim() == 3, "q must be [batch, num_heads, head_dim]")
    batch, num_heads, head_dim = q.shape
    _, kvh, psize, hd = _check_pool(q, k_pool, v_pool, page_table, seq_lens, num_heads, check_tables)
    _req(hd == head_dim and page_table.shape[0] == batch and seq_lens.shape == (batch,), "shape mismatch")
    max_pages = page_table.shape[1]
    out = torch.empty_like(q) if out is None else out
    _cuda(out, "out")
    _req(out.shape == q.shape and out.dtype == q.dtype, "out must match q")
    if workspace is None:
        workspace = attention_workspace(batch, num_heads, head_dim, max_pages * psize, q.device)
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    hip.call("cir_paged_decode_attention", q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), page_table.data_ptr(),
             seq_lens.data_ptr(), out.data_ptr(), workspace.data_ptr(), workspace.numel(), batch, num_heads, kvh,
             head_dim, psize, max_pages, float(scale), hip.dtype_code(q.dtype), hip.stream_handle())
    return out


def paged_decode_attention_noalloc(q, k_pool, v_pool, page_table, seq_lens, *, scale: float | None = None,
                                   out: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_decode_attention`` through ``cir_paged_decode_attention_noalloc``: the split partials go to the
    library's static per-GPU scratch (no workspace; calls overlapping on one GPU race).  ``out`` must be given by
    callers that cannot allocate."""
    _req(q.dim() == 3, "q must be [batch, num_heads, head_dim]")
    batch, num_heads, head_dim = q.shape
    _, kvh, psize, hd = _check_pool(q, k_pool, v_pool, page_table, seq_lens, num_heads, False)
    _req(hd == head_dim and page_table.shape[0] == batch and seq_lens.shape == (batch,), "shape mismatch")
    out = torch.empty_like(q) if out is None else out
    _cuda(out, "out")
    _req(out.shape == q.shape and out.dtype == q.dtype, "out must match q")
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    hip.call("cir_paged_decode_attention_noalloc", q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
             page_table.data_ptr(), seq_lens.data_ptr(), out.data_ptr(), batch, num_heads, kvh, head_dim, psize,
             page_table.shape[1], float(scale), hip.dtype_code(q.dtype), hip.stream_handle())
    return out


def paged_decode_attention_qkv(part, inv_freq, positions, k_pool, v_pool, page_table, seq_lens, *, num_heads: int,
                               scale: float | None = None, out: torch.Tensor | None = None,
                               workspace: torch.Tensor | None = None, check_tables: bool = False) -> torch.Tensor:
    """Decode attention fed by the QKV projection's fp32 partials ``[splits, B, (Hq + 2 Hkv) D]``: RoPE, the KV
    append of the new token and attention in one launch (fp16 pools, head_dim 128). Returns out ``[B, Hq, D]``."""
    _cuda(part, "part")
    _req(part.dtype == torch.float32 and part.dim() == 3, "part must be float32 [splits, batch, n]", TypeError)
    splits, batch, n = part.shape
    _req(k_pool.dtype == torch.float16, "the fused QKV attention needs float16 pools", TypeError)
    _, kvh, psize, hd = _check_pool(k_pool, k_pool, v_pool, page_table, seq_lens, num_heads, check_tables)
    _req(n == (num_heads + 2 * kvh) * hd, "qkv partial width must be (num_heads + 2 kv_heads) * head_dim")
    _req(page_table.shape[0] == batch and seq_lens.shape == (batch,), "shape mismatch")
    _cuda(positions, "positions")
    _cuda(inv_freq, "inv_freq")
    _req(positions.dtype == torch.int32 and positions.numel() == batch, "positions must be int32 [batch]", TypeError)
    _req(inv_freq.dtype == torch.float32 and inv_freq.numel() == hd // 2, "inv_freq must be float32 [D/2]", TypeError)
    max_pages = page_table.shape[1]
    if out is None:
        out = torch.empty((batch, num_heads, hd), dtype=k_pool.dtype, device=k_pool.device)
    _cuda(out, "out")
    _req(out.shape == (batch, num_heads, hd) and out.dtype == k_pool.dtype, "out must be [batch, num_heads, head_dim]")
    if workspace is None:
        workspace = attention_workspace(batch, num_heads, hd, max_pages * psize, k_pool.device)
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    hip.call("cir_paged_decode_attention_qkv", part.data_ptr(), splits, inv_freq.data_ptr(), positions.data_ptr(),
             k_pool.data_ptr(), v_pool.data_ptr(), page_table.data_ptr(), seq_lens.data_ptr(), out.data_ptr(),
             workspace.data_ptr(), workspace.numel(), batch, num_heads, kvh, hd, psize, max_pages, float(scale),
             hip.stream_handle())
    return out


def paged_prefill_attention(q, k_pool, v_pool, page_table, seq_lens, q_len: int, *, scale: float | None = None,
                            out=None, workspace=None, check_tables: bool = False,
                            own_workspace: bool = False) -> torch.Tensor:
    """q ``[B*q_len, Hq, D]``; ``seq_lens`` are lengths after appending the q_len tokens (causal).  A few queries over
    a long context run as context splits; their partials go to a buffer of this call, or to ``workspace`` if
    ``own_workspace`` says that no other launch uses it meanwhile (a workspace is otherwise not written on the fp16
    head_dim-128 path, so overlapping prefills may share one)."""
    _req(q.dim() == 3 and q_len >= 1 and q.shape[0] % q_len == 0, "q must be [batch*q_len, num_heads, head_dim]")
    rows, num_heads, head_dim = q.shape
    batch = rows // q_len
    _, kvh, psize, hd = _check_pool(q, k_pool, v_pool, page_table, seq_lens, num_heads, check_tables)
    _req(hd == head_dim and page_table.shape[0] == batch and seq_lens.shape == (batch,), "shape mismatch")
    max_pages = page_table.shape[1]
    out = torch.empty_like(q) if out is None else out
    code = hip.dtype_code(q.dtype)
    if workspace is None:
        workspace = attention_workspace(rows, num_heads, head_dim, max_pages * psize, q.device)
        own_workspace = True
    name = "cir_paged_prefill_attention_split"  # (it takes any sizes, and the advertised workspace holds its partials)
    if not own_workspace:
        need = hip.size_call("cir_paged_prefill_split_bytes", batch, q_len, num_heads, kvh, head_dim, psize, max_pages, code)
        if need:
            _req(workspace.numel() >= hip.size_call("cir_paged_attention_workspace_bytes", rows, num_heads, head_dim,
                                                    max_pages * psize), "attention: workspace too small", RuntimeError)
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        else:
            name = "cir_paged_prefill_attention"
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    hip.call(name, q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), page_table.data_ptr(), seq_lens.data_ptr(),
             out.data_ptr(), workspace.data_ptr(), workspace.numel(), batch, q_len, num_heads, kvh, head_dim, psize,
             max_pages, float(scale), code, hip.stream_handle())
    return out


def shared_attention_workspace(batch: int, groups: int, num_heads: int, num_kv_heads: int, head_dim: int,
                               page_size: int, max_pages: int, kv_dtype: torch.dtype, device) -> torch.Tensor:
    """Workspace of ``paged_decode_attention_shared`` at these sizes (one per call that may overlap another)."""
    n = hip.size_call("cir_shared_attention_workspace_bytes", batch, groups, num_heads, num_kv_heads, head_dim, page_size,
                      max_pages, hip.dtype_code(kv_dtype))
    return torch.empty(max(n, 4), dtype=torch.uint8, device=device)


def _check_workspace(workspace, dev: int) -> None:
    if not (workspace.get_device() == dev and workspace.is_contiguous()):
        _cuda(workspace, "workspace")
        _req(False, f"workspace must be on cuda:{dev}")


def _check_shared(q, k_pool, v_pool, page_table, seq_lens, group_rows, prefix_lens, check_tables: bool) -> None:
    for t, n in ((q, "q"), (k_pool, "k_pool"), (group_rows, "group_rows"), (prefix_lens, "prefix_lens")):
        _cuda(t, n)
    _req(q.dim() == 3, "q must be [batch, num_heads, head_dim]")
    batch, num_heads, head_dim = q.shape
    _, _, psize, hd = _check_pool(q, k_pool, v_pool, page_table, seq_lens, num_heads, check_tables)
    _req(hd == head_dim and page_table.dim() == 2 and page_table.shape[0] == batch and seq_lens.shape == (batch,),
         "shape mismatch")
    groups, max_pages = prefix_lens.numel(), page_table.shape[1]
    _tensors(q.device, k_pool=(k_pool, q.dtype, k_pool.shape), v_pool=(v_pool, q.dtype, k_pool.shape),
             page_table=(page_table, torch.int32, page_table.shape), seq_lens=(seq_lens, torch.int32, (batch,)),
             group_rows=(group_rows, torch.int32, (groups + 1,)), prefix_lens=(prefix_lens, torch.int32, (groups,)))
    if check_tables:
        rows, lens, table = group_rows.tolist(), prefix_lens.tolist(), page_table.cpu()
        _req(all(a <= b for a, b in zip(rows, rows[1:])) and 0 <= rows[0] and rows[-1] <= batch,
             "group_rows must ascend within the batch")
        for g, n in enumerate(lens):
            part = table[rows[g]: rows[g + 1], : -(-max(0, n) // psize)]  # the page it ends in too
            _req(0 <= n <= max_pages * psize, "prefix_lens exceed the page table capacity")
            _req(part.numel() == 0 or bool((part == part[:1]).all()), f"group {g}: rows with other pages in the prefix")


def paged_decode_attention_shared(q, k_pool, v_pool, page_table, seq_lens, group_rows, prefix_lens, *,
                                  scale: float | None = None, out: torch.Tensor | None = None,
                                  workspace: torch.Tensor | None = None, check_tables: bool = False) -> torch.Tensor:
    """``paged_decode_attention`` of a batch whose rows share prefixes: rows ``group_rows[g] .. group_rows[g + 1] - 1``
    (int32 ``[groups + 1]``, ascending) have the same pages for their first ``prefix_lens[g]`` tokens (int32
    ``[groups]``; the page in which they end is the same too), and each prefix is read once for all of them.  Both may
    change between replays of a captured call.  ``check_tables`` checks them, the pages and the lengths on the host (a
    device sync)."""
    dev, dt = q.get_device(), q.dtype
    qs, ps, ts, i32 = q.shape, k_pool.shape, page_table.shape, torch.int32
    groups = prefix_lens.numel()
    if not (dev >= 0 and len(qs) == 3 and len(ps) == 4 and len(ts) == 2 and not check_tables
            and qs[0] == ts[0] and qs[2] == ps[3] and _fits(q, dev, dt, qs) and _fits(k_pool, dev, dt, ps)
            and _fits(v_pool, dev, dt, ps) and _fits(page_table, dev, i32, ts) and _fits(seq_lens, dev, i32, qs[:1])
            and _fits(prefix_lens, dev, i32, (groups,)) and _fits(group_rows, dev, i32, (groups + 1,))):
        _check_shared(q, k_pool, v_pool, page_table, seq_lens, group_rows, prefix_lens, check_tables)
    batch, num_heads, head_dim = qs
    _, kvh, psize, _ = ps
    max_pages = ts[1]
    _int32(batch, num_heads, kvh, head_dim, psize, max_pages, groups)
    if out is None:
        out = torch.empty_like(q)
    elif not _fits(out, dev, dt, q.shape):
        _tensors(q.device, out=(out, dt, q.shape))
    if batch == 0:
        return out
    if workspace is None:
        workspace = shared_attention_workspace(batch, groups, num_heads, kvh, head_dim, psize, max_pages, q.dtype,
                                               q.device)
    _check_workspace(workspace, dev)
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    _call_on(dev, "cir_paged_decode_attention_shared", q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
             page_table.data_ptr(), seq_lens.data_ptr(), group_rows.data_ptr(), prefix_lens.data_ptr(), groups,
             out.data_ptr(), workspace.data_ptr(), workspace.nbytes, batch, num_heads, kvh, head_dim, psize, max_pages,
             scale, hip.dtype_code(dt))
    return out


def tree_attention_workspace(tokens: int, batch: int, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int,
                             max_pages: int, kv_dtype: torch.dtype, device) -> torch.Tensor:
    """Workspace of ``paged_tree_attention`` at these sizes (one per call that may overlap another)."""
    n = hip.size_call("cir_tree_attention_workspace_bytes", tokens, batch, num_heads, num_kv_heads, head_dim, page_size,
                      max_pages, hip.dtype_code(kv_dtype))
    return torch.empty(max(n, 4), dtype=torch.uint8, device=device)


def _check_tree(q, k_pool, v_pool, page_table, seq_lens, offsets, counts, masks, check_tables: bool) -> None:
    for t, n in ((q, "q"), (k_pool, "k_pool"), (masks, "masks")):
        _cuda(t, n)
    _req(q.dim() == 3, "q must be [tokens, num_heads, head_dim]")
    tokens, num_heads, head_dim = q.shape
    _, _, psize, hd = _check_pool(q, k_pool, v_pool, page_table, seq_lens, num_heads, False)
    _req(hd == head_dim and page_table.dim() == 2, "shape mismatch")
    _req(masks.dim() == 2 and masks.shape[0] == tokens, "masks must be [tokens, words]")
    batch, max_pages = page_table.shape
    _tensors(q.device, k_pool=(k_pool, q.dtype, k_pool.shape), v_pool=(v_pool, q.dtype, k_pool.shape),
             page_table=(page_table, torch.int32, page_table.shape), seq_lens=(seq_lens, torch.int32, (batch,)),
             offsets=(offsets, torch.int32, (batch + 1,)), counts=(counts, torch.int32, (batch,)),
             masks=(masks, torch.int64, masks.shape))
    if check_tables:
        at, n, lens, table = offsets.tolist(), counts.tolist(), seq_lens.tolist(), page_table.cpu()
        _req(all(a <= b for a, b in zip(at, at[1:])) and 0 <= at[0] and at[-1] <= tokens,
             "offsets must ascend within the tokens")
        for b in range(batch):
            _req(0 <= n[b] <= min(at[b + 1] - at[b], 64 * masks.shape[1], lens[b]),
                 f"row {b}: counts exceed its tokens, the masks or its length")
            _req(lens[b] <= max_pages * psize, "seq_lens exceed the page table capacity")
            used = table[b, : -(-lens[b] // psize)]
            _req(used.numel() == 0 or (int(used.min()) >= 0 and int(used.max()) < k_pool.shape[0]),
                 "page_table has slots outside the pool")


def paged_tree_attention(q, k_pool, v_pool, page_table, seq_lens, offsets, counts, masks, *, scale: float | None = None,
                         out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                         check_tables: bool = False) -> torch.Tensor:
    """Attention of drafted tokens q ``[T, Hq, D]``: row b's are ``q[offsets[b] : offsets[b] + counts[b]]`` (int32
    ``[B + 1]``, ``[B]``; ``StepTables.offsets`` and ``.granted``), the last of its ``seq_lens[b]`` tokens in the pages.
    Each sees the tokens before the drafted ones, and drafted token k of its row where bit k % 64 of its
    ``masks[:, k // 64]`` (int64 ``[T, words]``, ``draft_tree``) is set.  Rows of q that no row counts keep their ``out``;
    all of a row of more tokens than its masks have bits for become NaN.
    ``check_tables`` checks lengths, offsets and pages on the host (a device sync)."""
    dev, dt, i32 = q.get_device(), q.dtype, torch.int32
    qs, ps, ts, ms = q.shape, k_pool.shape, page_table.shape, masks.shape
    if not (dev >= 0 and len(qs) == 3 and len(ps) == 4 and len(ts) == 2 and len(ms) == 2 and not check_tables
            and qs[2] == ps[3] and ms[0] == qs[0] and _fits(q, dev, dt, qs) and _fits(k_pool, dev, dt, ps)
            and _fits(v_pool, dev, dt, ps) and _fits(page_table, dev, i32, ts) and _fits(seq_lens, dev, i32, ts[:1])
            and _fits(offsets, dev, i32, (ts[0] + 1,)) and _fits(counts, dev, i32, ts[:1])
            and _fits(masks, dev, torch.int64, ms)):
        _check_tree(q, k_pool, v_pool, page_table, seq_lens, offsets, counts, masks, check_tables)
    tokens, num_heads, head_dim = qs
    _, kvh, psize, _ = ps
    batch, max_pages = ts
    words = ms[1]
    _int32(tokens, num_heads, kvh, head_dim, psize, batch, max_pages, words)
    code = hip.dtype_code(dt)
    if out is None:
        out = torch.empty_like(q)
    elif not _fits(out, dev, dt, qs):
        _tensors(q.device, out=(out, dt, qs))
    if workspace is None:
        n = hip.size_call("cir_tree_attention_workspace_bytes", tokens, batch, num_heads, kvh, head_dim, psize, max_pages,
                          code)
        workspace = torch.empty(max(n, 4), dtype=torch.uint8, device=q.device)
    else:
        _check_workspace(workspace, dev)
    _call_on(dev, "cir_paged_tree_attention", q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), page_table.data_ptr(),
             seq_lens.data_ptr(), offsets.data_ptr(), counts.data_ptr(), masks.data_ptr(), words, out.data_ptr(),
             workspace.data_ptr(), workspace.nbytes, tokens, batch, num_heads, kvh, head_dim, psize, max_pages,
             1.0 / math.sqrt(head_dim) if scale is None else scale, code)
    return out


# ---------------------------------------------------------------- step inputs --
class StepTables(NamedTuple):
    """What ``extend_page_tables`` writes beside the page table (see ``cir_extend_page_tables``)."""

    seq_lens: torch.Tensor   # int32 [batch]: lengths with the granted tokens
    free_head: torch.Tensor  # int32 [1]: first free slot not taken
    offsets: torch.Tensor    # int32 [batch + 1]: where each row's new tokens begin
    positions: torch.Tensor  # int32 [max_tokens]
    slot_map: torch.Tensor   # int64 [max_tokens]: place in the pools, -1 where there is none
    granted: torch.Tensor    # int32 [batch]: new tokens that got their pages (all of a row's or none)

    @classmethod
    def empty(cls, batch: int, max_tokens: int, device) -> "StepTables":
        # one allocation for what is int32 (six of them took 8 us of a call)
        lens, head, offsets, positions, granted = torch.empty(
            3 * batch + 2 + max_tokens, dtype=torch.int32, device=device).split_with_sizes(
                (batch, 1, batch + 1, max_tokens, batch))
        return cls(lens, head, offsets, positions, torch.empty(max_tokens, dtype=torch.int64, device=device), granted)


def extend_page_tables(page_table: torch.Tensor, seq_lens: torch.Tensor, new_tokens: torch.Tensor,
                       free_slots: torch.Tensor, free_head: torch.Tensor, *, page_size: int, max_tokens: int,
                       out: StepTables | None = None) -> StepTables:
    """Page tables, positions and slot maps of a step on the GPU: row b's ``new_tokens[b]`` tokens after its
    ``seq_lens[b]``, new pages taken from ``free_slots[free_head:]`` in row order and written into ``page_table``.
    ``max_tokens`` bounds the new tokens of all rows (the map's length; its tail is -1).  ``out`` may hold ``seq_lens``
    and ``free_head`` themselves, which then advance in place (a captured decode step replays without the host)."""
    dev, i32 = page_table.get_device(), torch.int32
    shape, rows = page_table.shape, page_table.shape[:1]
    if not (dev >= 0 and len(shape) == 2 and _fits(page_table, dev, i32, shape) and _fits(seq_lens, dev, i32, rows)
            and _fits(new_tokens, dev, i32, rows) and _fits(free_slots, dev, i32, (free_slots.numel(),))
            and _fits(free_head, dev, i32, (1,))):
        _cuda(page_table, "page_table")
        _req(page_table.dim() == 2, "page_table must be [batch, pages]")
        _cuda(free_slots, "free_slots")
        _tensors(page_table.device, page_table=(page_table, i32, page_table.shape),
                 seq_lens=(seq_lens, i32, page_table.shape[:1]), new_tokens=(new_tokens, i32, page_table.shape[:1]),
                 free_slots=(free_slots, i32, (free_slots.numel(),)), free_head=(free_head, i32, (1,)))
    batch, max_pages = shape
    _req(page_size > 0 and max_tokens >= 0, "page_size must be positive and max_tokens not negative")
    _int32(batch, max_pages, page_size, max_tokens, free_slots.numel())
    if out is None:
        out = StepTables.empty(batch, max_tokens, page_table.device)
    else:
        _tensors(page_table.device, **{
            "out.seq_lens": (out.seq_lens, i32, (batch,)), "out.free_head": (out.free_head, i32, (1,)),
            "out.offsets": (out.offsets, i32, (batch + 1,)), "out.positions": (out.positions, i32, (max_tokens,)),
            "out.slot_map": (out.slot_map, torch.int64, (max_tokens,)), "out.granted": (out.granted, i32, (batch,))})
    lens, head, offsets, positions, slot_map, granted = out
    _call_on(dev, "cir_extend_page_tables", page_table.data_ptr(), seq_lens.data_ptr(), new_tokens.data_ptr(),
             free_slots.data_ptr(), free_slots.numel(), free_head.data_ptr(), lens.data_ptr(), head.data_ptr(),
             offsets.data_ptr(), granted.data_ptr(), positions.data_ptr(), slot_map.data_ptr(), batch, max_pages,
             page_size, max_tokens)
    return out


def rope_frequencies(rotary_dim: int, theta: float, scaling: dict | None = None, device="cuda") -> torch.Tensor:
    """Angles per position of the ``rotary_dim / 2`` pairs, ``theta ** (-2 i / rotary_dim)`` in float64, for
    ``rope_append``.  ``scaling`` as model configurations write it: ``{"rope_type": "linear", "factor": s}`` divides
    every frequency by s; ``"llama3"`` (with ``low_freq_factor`` a, ``high_freq_factor`` b and
    ``original_max_position_embeddings`` n) keeps frequencies of more than b turns in n positions, divides those of
    fewer than a by the factor and passes from one to the other linearly in the number of turns.  Other schemes: pass
    their own table (and their factor on cos and sin) to ``rope_append``."""
    _req(rotary_dim >= 0 and rotary_dim % 2 == 0, "rotary_dim must be even")
    _req(theta > 0, "theta must be positive")
    f = theta ** (-2.0 * torch.arange(rotary_dim // 2, dtype=torch.float64) / max(rotary_dim, 1))
    kind = (scaling or {}).get("rope_type", (scaling or {}).get("type", "default"))
    if kind == "linear":
        f = f / float(scaling["factor"])
    elif kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        _req(high > low, "high_freq_factor must exceed low_freq_factor")
        turns = f * float(scaling["original_max_position_embeddings"]) / (2.0 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        f = keep * f + (1.0 - keep) * f / float(scaling["factor"])
    else:
        _req(kind == "default", f"unsupported rope scaling {kind!r}")
    return f.to(device)


def _check_rope(q, k, v, positions, slot_map, inv_freq, k_pool, v_pool) -> None:
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _req(isinstance(t, torch.Tensor), f"{n} must be a torch.Tensor", TypeError)
        _req(t.is_cuda and t.device == q.device, f"{n} must be on the GPU, with q")
        _req(t.dim() == 3 and (t.stride(2) == 1 or t.shape[2] == 1),
             f"{n} must be [tokens, heads, head_dim] with contiguous heads")
        _req(t.dtype == q.dtype, "q, k and v must share a dtype", TypeError)
    tokens, _, dim = q.shape
    kvh = k.shape[1]
    _req(k.shape == v.shape == (tokens, kvh, dim), "k and v must be [tokens, kv_heads, head_dim] of q's tokens and dims")
    _cuda(k_pool, "k_pool")
    _req(k_pool.dim() == 4 and k_pool.shape[1] == kvh and k_pool.shape[3] == dim,
         "pools must be [slots, kv_heads, page_size, head_dim] of k's heads")
    _cuda(inv_freq, "inv_freq")
    _tensors(q.device, k_pool=(k_pool, k_pool.dtype, k_pool.shape), v_pool=(v_pool, k_pool.dtype, k_pool.shape),
             positions=(positions, torch.int32, (tokens,)), slot_map=(slot_map, torch.int64, (tokens,)),
             inv_freq=(inv_freq, torch.float64, (inv_freq.numel(),)))
    _req(2 * inv_freq.numel() <= dim, f"inv_freq turns {2 * inv_freq.numel()} dims of heads of {dim}")


def _rope_call(name: str, q, k, v, norm: tuple, positions, slot_map, inv_freq, k_pool, v_pool, layout: str,
               factor: float, out: torch.Tensor | None) -> torch.Tensor:
    """The checks and the call of ``rope_append`` and ``norm_rope_append`` (``norm``: the latter's arguments)."""
    dev, dt, kdt = q.get_device(), q.dtype, k_pool.dtype
    qs, ks, ps, fs = q.shape, k.shape, k_pool.shape, inv_freq.shape
    qt, kt, vt = q.stride(), k.stride(), v.stride()
    if not (dev >= 0 and len(qs) == len(ks) == 3 and len(ps) == 4 and len(fs) == 1
            and k.get_device() == dev == v.get_device() and k.dtype is dt is v.dtype and v.shape == ks
            and qs[0] == ks[0] and ps[3] == qs[2] == ks[2] >= 2 * fs[0] and ps[1] == ks[1]
            and qt[2] == kt[2] == vt[2] == 1
            and _fits(k_pool, dev, kdt, ps) and _fits(v_pool, dev, kdt, ps) and _fits(positions, dev, torch.int32, qs[:1])
            and _fits(slot_map, dev, torch.int64, qs[:1]) and _fits(inv_freq, dev, torch.float64, fs)):
        _check_rope(q, k, v, positions, slot_map, inv_freq, k_pool, v_pool)
    if layout not in hip.ROPE_LAYOUTS:
        _req(False, f"layout must be one of {sorted(hip.ROPE_LAYOUTS)}")
    tokens, heads, dim = qs
    slots, kvh, psize, _ = ps
    _int32(tokens, heads, kvh, dim, psize)
    if out is None:
        out = q.new_empty(qs)
        ot = (heads * dim, dim)
    else:
        _req(isinstance(out, torch.Tensor) and out.device == q.device and out.shape == q.shape and
             (out.stride(2) == 1 or dim == 1) and out.dtype == dt, "out must be like q")
        ot = out.stride()
    _call_on(dev, name, q.data_ptr(), qt[0], qt[1], k.data_ptr(), kt[0], kt[1], v.data_ptr(), vt[0], vt[1],
             hip.dtype_code(dt), *norm, positions.data_ptr(), slot_map.data_ptr(), inv_freq.data_ptr(), factor, 2 * fs[0],
             hip.ROPE_LAYOUTS[layout], out.data_ptr(), ot[0], ot[1], k_pool.data_ptr(), v_pool.data_ptr(),
             hip.dtype_code(kdt), slots * psize, tokens, heads, kvh, dim, psize)
    return out


def rope_append(q, k, v, positions, slot_map, inv_freq, k_pool, v_pool, *, layout: str = "interleaved",
                factor: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions of q ``[T, Hq, D]`` and k ``[T, Hkv, D]`` at ``positions`` and the append of k and v to the pools
    at ``slot_map`` (int64, a token's page * page_size + offset; outside the pools: padding, nothing is written).  The
    first ``2 * inv_freq.numel()`` dims of a head turn, in pairs (2i, 2i + 1) (``"interleaved"``) or halves apart
    (``"half"``); cos and sin are multiplied by ``factor``.  q, k and v may be views (any token and head stride, as the
    columns of one QKV projection); ``out`` may be q, and otherwise overlaps no input.  Returns the turned q."""
    return _rope_call("cir_rope_append", q, k, v, (), positions, slot_map, inv_freq, k_pool, v_pool, layout, factor, out)


def norm_rope_append(q, k, v, q_weight, k_weight, eps: float, positions, slot_map, inv_freq, k_pool, v_pool, *,
                     layout: str = "interleaved", factor: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """``rope_append`` with an RMS norm of each head of q and k before it turns: ``x / sqrt(mean(x ** 2) + eps) *
    weight``, ``q_weight`` and ``k_weight`` ``[head_dim]`` (float32 or float16).  Rounded once, to the output."""
    dev, wdt, shape = q.get_device(), q_weight.dtype, q.shape[-1:]
    if not (dev >= 0 and _fits(q_weight, dev, wdt, shape) and _fits(k_weight, dev, wdt, shape)):
        _cuda(q, "q") if dev < 0 else None
        _tensors(q.device, q_weight=(q_weight, wdt, shape), k_weight=(k_weight, wdt, shape))
    return _rope_call("cir_norm_rope_append", q, k, v, (q_weight.data_ptr(), k_weight.data_ptr(), hip.dtype_code(wdt), eps),
                      positions, slot_map, inv_freq, k_pool, v_pool, layout, factor, out)


# -------------------------------------------------------------- drafted trees --
class DraftTree(NamedTuple):
    masks: torch.Tensor      # int64 [tokens, words]: bit k % 64 of word k / 64 where token k of the row is seen
    positions: torch.Tensor  # int32 [tokens]


def draft_tree(parents: torch.Tensor, seq_lens: torch.Tensor, offsets: torch.Tensor, counts: torch.Tensor, *, words: int,
               out: DraftTree | None = None) -> DraftTree:
    """What each drafted token sees of its row's tree (itself and its ancestors) and its rotary position, from
    ``parents`` (int32 ``[T]``, places in the row's tree, negative: it follows the context).  Row b's tokens are
    ``offsets[b] .. offsets[b] + counts[b] - 1``, up to ``64 * words`` (words 1..4; a row of more gets empty masks), and the
    last of its ``seq_lens[b]``; see ``cir_draft_tree``."""
    dev, i32 = parents.get_device(), torch.int32
    tokens, batch = parents.numel(), counts.numel()
    if not (dev >= 0 and _fits(parents, dev, i32, (tokens,)) and _fits(counts, dev, i32, (batch,))
            and _fits(seq_lens, dev, i32, (batch,)) and _fits(offsets, dev, i32, (batch + 1,))):
        _cuda(parents, "parents")
        _tensors(parents.device, parents=(parents, i32, (tokens,)), counts=(counts, i32, (batch,)),
                 seq_lens=(seq_lens, i32, (batch,)), offsets=(offsets, i32, (batch + 1,)))
    _req(1 <= words <= 4, f"words must be 1..4 (got {words})")
    _int32(tokens, batch)
    if out is None:
        out = DraftTree(torch.empty((tokens, words), dtype=torch.int64, device=parents.device),
                        torch.empty(tokens, dtype=i32, device=parents.device))
    else:
        _tensors(parents.device, **{"out.masks": (out.masks, torch.int64, (tokens, words)),
                                    "out.positions": (out.positions, i32, (tokens,))})
    _call_on(dev, "cir_draft_tree", parents.data_ptr(), seq_lens.data_ptr(), offsets.data_ptr(), counts.data_ptr(),
             out.masks.data_ptr(), out.positions.data_ptr(), tokens, batch, words)
    return out


class AcceptedDrafts(NamedTuple):
    accepted: torch.Tensor  # int32 [batch]: drafted tokens that stand, and so tokens said
    path: torch.Tensor      # int32 [batch, most]: their places in the row's tree, then -1
    tokens: torch.Tensor    # int64 [batch, most]: what the model chose after each, then -1
    seq_lens: torch.Tensor  # int32 [batch]: lengths with them

    @classmethod
    def empty(cls, batch: int, most: int, device) -> "AcceptedDrafts":
        # one allocation for what is int32
        accepted, path, lens = torch.empty(batch * (most + 2), dtype=torch.int32,
                                           device=device).split_with_sizes((batch, batch * most, batch))
        return cls(accepted, path.view(batch, most), torch.empty((batch, most), dtype=torch.int64, device=device), lens)


def accept_drafts(parents: torch.Tensor, drafts: torch.Tensor, targets: torch.Tensor, seq_lens: torch.Tensor,
                  offsets: torch.Tensor, counts: torch.Tensor, page_table: torch.Tensor, k_pools: torch.Tensor,
                  v_pools: torch.Tensor, *, most: int, free_slots: torch.Tensor | None = None,
                  free_head: torch.Tensor | None = None, out: AcceptedDrafts | None = None) -> AcceptedDrafts:
    """The drafted tokens that the model's choices confirm: from the row's token 0 on, the child whose ``drafts`` (int64
    ``[T]``) equals ``targets`` (int64 ``[T]``, chosen after each token), ``most`` tokens at most, none past the row's
    first 256.  K and V of the path move behind the context in the pools of all layers (``[layers, slots, kv_heads, page_size, head_dim]``).  With
    ``free_slots`` and ``free_head`` (as ``extend_page_tables`` takes them) pages behind the new lengths go back.
    ``out.seq_lens`` may be ``seq_lens``.  See ``cir_accept_drafts``."""
    dev, i32, i64 = parents.get_device(), torch.int32, torch.int64
    tokens, ts, ps, dt = parents.numel(), page_table.shape, k_pools.shape, k_pools.dtype
    rows = ts[:1]
    if not (dev >= 0 and len(ts) == 2 and len(ps) == 5 and _fits(parents, dev, i32, (tokens,))
            and _fits(drafts, dev, i64, (tokens,)) and _fits(targets, dev, i64, (tokens,))
            and _fits(seq_lens, dev, i32, rows) and _fits(counts, dev, i32, rows)
            and _fits(offsets, dev, i32, (ts[0] + 1,)) and _fits(page_table, dev, i32, ts)
            and _fits(k_pools, dev, dt, ps) and _fits(v_pools, dev, dt, ps)):
        _cuda(parents, "parents")
        _req(page_table.dim() == 2, "page_table must be [batch, pages]")
        _req(k_pools.dim() == 5, "pools must be [layers, slots, kv_heads, page_size, head_dim]")
        _tensors(parents.device, parents=(parents, i32, (tokens,)), drafts=(drafts, i64, (tokens,)),
                 targets=(targets, i64, (tokens,)), seq_lens=(seq_lens, i32, rows), counts=(counts, i32, rows),
                 offsets=(offsets, i32, (ts[0] + 1,)), page_table=(page_table, i32, ts), k_pools=(k_pools, dt, ps),
                 v_pools=(v_pools, dt, ps))
    batch, max_pages = ts
    layers, slots, kvh, psize, head_dim = ps
    _req(1 <= most <= 256, f"most must be 1..256 (got {most})")
    _int32(tokens, batch, max_pages, layers, kvh, psize, head_dim)
    _req((free_slots is None) == (free_head is None), "free_slots and free_head go together")
    total = 0
    if free_slots is not None:
        total = free_slots.numel()
        _tensors(parents.device, free_slots=(free_slots, i32, (total,)), free_head=(free_head, i32, (1,)))
        _int32(total)
    if out is None:
        out = AcceptedDrafts.empty(batch, most, parents.device)
    else:
        _tensors(parents.device, **{"out.accepted": (out.accepted, i32, rows), "out.path": (out.path, i32, (batch, most)),
                                    "out.tokens": (out.tokens, i64, (batch, most)), "out.seq_lens": (out.seq_lens, i32, rows)})
    _call_on(dev, "cir_accept_drafts", parents.data_ptr(), drafts.data_ptr(), targets.data_ptr(), seq_lens.data_ptr(),
             offsets.data_ptr(), counts.data_ptr(), page_table.data_ptr(), out.accepted.data_ptr(), out.path.data_ptr(),
             out.tokens.data_ptr(), out.seq_lens.data_ptr(), k_pools.data_ptr(), v_pools.data_ptr(), hip.dtype_code(dt),
             slots, hip.ptr(free_slots), total, hip.ptr(free_head), tokens, batch, most, max_pages, layers, kvh, head_dim,
             psize)
    return out


# -------------------------------------------------------------- block weights --
@dataclass
class QWeight:
    """A Q4_0/Q8_0 (or per-row asymmetric int4/int8) weight ``W[n, k]`` kept on the device in the tiled layout."""

    tiled: torch.Tensor  # uint8
    fmt: int
    n: int
    k: int

    @property
    def shape(self) -> tuple[int, int]:
        return (self.n, self.k)

    @property
    def nbytes(self) -> int:
        return self.tiled.numel()

    @classmethod
    def from_rows(cls, packed: torch.Tensor, scales: torch.Tensor, zero_points: torch.Tensor, bits: int, n: int,
                  k: int) -> "QWeight":
        """Repack the reference's per-row asymmetric packing (uint8 codes ``[n, ceil(k/2)]`` for 4 bit or
        ``[n, k]`` for 8 bit, fp32 scales ``[n]``, int32 zero points ``[n]``, on the GPU) into the tiled layout."""
        for t, name in ((packed, "packed"), (scales, "scales"), (zero_points, "zero_points")):
            _cuda(t, name)
        _req(bits in (4, 8), f"bits must be 4 or 8 (got {bits})")
        _req(k % 128 == 0, f"k={k} must be a multiple of 128 for the tiled GEMM")
        row_bytes = (k + 1) // 2 if bits == 4 else k
        _req(packed.dtype == torch.uint8 and packed.numel() == n * row_bytes, "packed codes must be uint8 [n, row_bytes]")
        _req(scales.dtype == torch.float32 and scales.numel() == n, "scales must be float32 [n]", TypeError)
        _req(zero_points.dtype == torch.int32 and zero_points.numel() == n, "zero_points must be int32 [n]", TypeError)
        fmt = hip.CIR_I4_ROW if bits == 4 else hip.CIR_I8_ROW
        size = hip.size_call("cir_qweight_tiled_bytes", fmt, n, k)
        tiled = torch.empty(size, dtype=torch.uint8, device=packed.device)
        hip.call("cir_qweight_repack_rows", packed.data_ptr(), scales.data_ptr(), zero_points.data_ptr(),
                 tiled.data_ptr(), fmt, n, k, hip.stream_handle())
        return cls(tiled, fmt, n, k)

    @classmethod
    def from_blocks(cls, blocks: torch.Tensor, fmt: int, n: int, k: int) -> "QWeight":
        """Repack GGUF blocks (uint8, ``n * k/32 * block_bytes``, on the GPU) into the tiled layout."""
        _cuda(blocks, "blocks")
        _req(fmt in BLOCK_BYTES, f"unsupported block format {fmt}")
        _req(k % 128 == 0, f"k={k} must be a multiple of 128 for the tiled GEMM")
        _req(blocks.dtype == torch.uint8 and blocks.numel() == n * (k // QK) * BLOCK_BYTES[fmt],
             "blocks must be uint8 with n*k/32*block_bytes elements")
        size = hip.size_call("cir_qweight_tiled_bytes", fmt, n, k)
        tiled = torch.empty(size, dtype=torch.uint8, device=blocks.device)
        hip.call("cir_qweight_repack", blocks.data_ptr(), tiled.data_ptr(), fmt, n, k, hip.stream_handle())
        return cls(tiled, fmt, n, k)


def dequant_blocks(blocks: torch.Tensor, fmt: int, n: int, k: int) -> torch.Tensor:
    _cuda(blocks, "blocks")
    _req(blocks.numel() == n * (k // QK) * BLOCK_BYTES[fmt], "block byte count mismatch")
    out = torch.empty((n, k), dtype=torch.float32, device=blocks.device)
    hip.call("cir_dequant", blocks.data_ptr(), 0, fmt, out.data_ptr(), n, k, hip.stream_handle())
    return out


def dequant_tiled(w: QWeight) -> torch.Tensor:
    out = torch.empty((w.n, w.k), dtype=torch.float32, device=w.tiled.device)
    hip.call("cir_dequant", w.tiled.data_ptr(), 1, w.fmt, out.data_ptr(), w.n, w.k, hip.stream_handle())
    return out


def paged_decode_splits(batch: int, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int,
                        max_pages: int, kv_dtype: torch.dtype) -> int:
    """Context splits the decode attention uses at these sizes (``cir_paged_decode_splits``)."""
    return hip.load().cir_paged_decode_splits(batch, num_heads, num_kv_heads, head_dim, page_size, max_pages,
                                              hip.dtype_code(kv_dtype))


def paged_decode_attention_qkv_parts(part, inv_freq, positions, k_pool, v_pool, page_table, seq_lens, *,
                                     num_heads: int, workspace: torch.Tensor, scale: float | None = None) -> int:
    """``paged_decode_attention_qkv`` without the merge: the split partials stay in ``workspace`` (O
    ``[B, Hq, S, D]`` fp32 at its start, (max, sum) ``[B, Hq, S, 2]`` after it) for ``qgemm_attn``.
    Returns S (> 1 is required)."""
    _cuda(part, "part")
    _req(part.dtype == torch.float32 and part.dim() == 3, "part must be float32 [splits, batch, n]", TypeError)
    splits, batch, n = part.shape
    _req(k_pool.dtype == torch.float16, "the fused QKV attention needs float16 pools", TypeError)
    _, kvh, psize, hd = _check_pool(k_pool, k_pool, v_pool, page_table, seq_lens, num_heads, False)
    _req(n == (num_heads + 2 * kvh) * hd, "qkv partial width must be (num_heads + 2 kv_heads) * head_dim")
    _req(page_table.shape[0] == batch and seq_lens.shape == (batch,), "shape mismatch")
    _cuda(positions, "positions")
    _cuda(inv_freq, "inv_freq")
    _cuda(workspace, "workspace")
    max_pages = page_table.shape[1]
    S = paged_decode_splits(batch, num_heads, kvh, hd, psize, max_pages, k_pool.dtype)
    _req(S > 1, "the unmerged decode attention needs more than one context split")
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    hip.call("cir_paged_decode_attention_qkv_parts", part.data_ptr(), splits, inv_freq.data_ptr(),
             positions.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), page_table.data_ptr(), seq_lens.data_ptr(),
             workspace.data_ptr(), workspace.numel() * workspace.element_size(), batch, num_heads, kvh, hd, psize,
             max_pages, float(scale), hip.stream_handle())
    return S


def qgemm_attn(workspace: torch.Tensor, attn_splits: int, num_heads: int, w: QWeight, m: int,
               splits: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """fp32 partials ``[splits, m, n]`` of ``merge(attention partials) @ W^T`` (``cir_qgemm_attn``): the attention
    output of ``m`` rows, merged from ``workspace`` as ``paged_decode_attention_qkv_parts`` left it, is the input."""
    _cuda(workspace, "workspace")
    _req(w.k == num_heads * 128, "the O projection's k must be num_heads * 128")
    head_dim = 128
    o_floats = m * num_heads * attn_splits * head_dim
    _req(workspace.numel() * workspace.element_size() >= 4 * (o_floats + m * num_heads * attn_splits * 2),
         "workspace smaller than the attention partials")
    splits = choose_splits(m, w.n, w.k) if splits is None else splits
    if out is None:
        out = torch.empty((splits, m, w.n), dtype=torch.float32, device=workspace.device)
    _req(out.numel() >= splits * m * w.n and out.dtype == torch.float32, "partial buffer too small")
    base = workspace.data_ptr()
    hip.call("cir_qgemm_attn", base, base + 4 * o_floats, attn_splits, num_heads, w.tiled.data_ptr(), w.fmt,
             out.data_ptr(), m, w.n, w.k, splits, hip.stream_handle())
    return out.view(-1)[: splits * m * w.n].view(splits, m, w.n)


def gemm_plan(op: int, fmt: int, m: int, n: int, k: int, splits: int = 1) -> str:
    """Name of the kernel the library runs for this GEMM (``cir_qgemm_plan``; op = ``hip.GEMM_*``)."""
    return hip.load().cir_qgemm_plan(op, fmt, m, n, k, splits).decode()


def choose_splits(m: int, n: int, k: int) -> int:
    """k-split the library tunes ``cir_qgemm`` for at this shape (``cir_qgemm_splits``)."""
    s = hip.load().cir_qgemm_splits(m, n, k)
    _req(s > 0, f"no k-split for shape m={m} n={n} k={k} (k must be a positive multiple of 128)")
    return s


def qgemm_partial(x: torch.Tensor, w: QWeight, splits: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """fp32 partials ``[splits, m, n]`` of ``x[m, k] @ W[n, k]^T`` (x fp16, rows contiguous, any row stride)."""
    _cuda(x, "x", rows_only=True)
    _req(x.dtype == torch.float16, "qgemm activations must be float16", TypeError)
    _req(x.dim() == 2 and x.shape[1] == w.k, f"x must be [m, {w.k}]")
    _req(x.stride(1) == 1 and x.stride(0) >= w.k, "x rows must be contiguous (row stride >= k)")
    m = x.shape[0]
    splits = choose_splits(m, w.n, w.k) if splits is None else splits
    if out is None:
        out = torch.empty((splits, m, w.n), dtype=torch.float32, device=x.device)
    _req(out.numel() >= splits * m * w.n and out.dtype == torch.float32, "partial buffer too small")
    if x.data_ptr() % 16 and (w.k // 128) % splits:  # only the large-m kernel takes such splits, and it reads x by DMA
        x = x.clone(memory_format=torch.contiguous_format)
    hip.call("cir_qgemm", x.data_ptr(), x.stride(0), w.tiled.data_ptr(), w.fmt, out.data_ptr(), m, w.n, w.k, splits,
             hip.stream_handle())
    return out.view(-1)[: splits * m * w.n].view(splits, m, w.n)


def interleave_gate_up(gate_blocks: torch.Tensor, up_blocks: torch.Tensor, rows: int) -> torch.Tensor:
    """GGUF block rows of gate and up ([rows, row_bytes] each, uint8) -> [2*rows, row_bytes] in the order
    gate 16c..16c+15, up 16c..16c+15, c = 0, 1, ... (the tile pairing ``cir_qgemm_swiglu`` reads)."""
    _req(rows % 16 == 0, "gate/up rows must be a multiple of 16")
    g = gate_blocks.reshape(rows // 16, 1, 16, -1)
    u = up_blocks.reshape(rows // 16, 1, 16, -1)
    return torch.cat([g, u], dim=1).reshape(2 * rows, -1).contiguous()


def qgemm_swiglu(x: torch.Tensor, w: QWeight, out_dtype: torch.dtype = torch.float16, out=None) -> torch.Tensor:
    """``silu(x @ gate^T) * (x @ up^T)`` from the interleaved gate|up tiled weight (``interleave_gate_up``)."""
    _cuda(x, "x", rows_only=True)
    _req(x.dtype == torch.float16, "qgemm activations must be float16", TypeError)
    _req(x.dim() == 2 and x.shape[1] == w.k and w.n % 32 == 0, f"x must be [m, {w.k}] and n a multiple of 32")
    m, inter = x.shape[0], w.n // 2
    if out is None:
        out = torch.empty((m, inter), dtype=out_dtype, device=x.device)
    _req(out.shape == (m, inter) and out.is_contiguous(), "out must be [m, n/2] contiguous")
    hip.call("cir_qgemm_swiglu", x.data_ptr(), x.stride(0), w.tiled.data_ptr(), w.fmt, out.data_ptr(),
             hip.dtype_code(out.dtype), m, inter, w.k, hip.stream_handle())
    return out


def qgemm_argmax_workspace(m: int, n: int, device) -> torch.Tensor:
    return torch.empty(max(hip.size_call("cir_qgemm_argmax_workspace_bytes", m, n), 4), dtype=torch.uint8,
                       device=device)


def qgemm_argmax(x: torch.Tensor, w: QWeight, out=None, workspace=None) -> torch.Tensor:
    """Greedy ids ``argmax_j (x @ W^T)[r, j]`` without storing the logits (first index on ties, NaN as the
    maximum); equal to ``argmax(qgemm_partial(x, w, splits=1)[0])``."""
    _cuda(x, "x", rows_only=True)
    _req(x.dtype == torch.float16, "qgemm activations must be float16", TypeError)
    _req(x.dim() == 2 and x.shape[1] == w.k, f"x must be [m, {w.k}]")
    m = x.shape[0]
    if out is None:
        out = torch.empty(m, dtype=torch.int64, device=x.device)
    _req(out.dtype == torch.int64 and out.numel() == m and out.is_contiguous(), "out must be int64 [m]", TypeError)
    if workspace is None:
        workspace = qgemm_argmax_workspace(m, w.n, x.device)
    hip.call("cir_qgemm_argmax", x.data_ptr(), x.stride(0), w.tiled.data_ptr(), w.fmt, out.data_ptr(),
             workspace.data_ptr(), workspace.numel() * workspace.element_size(), m, w.n, w.k, hip.stream_handle())
    return out


def gemm_f32_partial(x: torch.Tensor, w: torch.Tensor, splits: int = 1, out=None) -> torch.Tensor:
    _cuda(x, "x")
    _cuda(w, "w")
    _req(x.dtype == torch.float32 and w.dtype == torch.float32, "gemm_f32 needs float32 x and w", TypeError)
    _req(x.dim() == 2 and w.dim() == 2 and x.shape[1] == w.shape[1], "x [m,k] and w [n,k] required")
    m, k = x.shape
    n = w.shape[0]
    if out is None:
        out = torch.empty((splits, m, n), dtype=torch.float32, device=x.device)
    hip.call("cir_gemm_f32", x.data_ptr(), k, w.data_ptr(), out.data_ptr(), m, n, k, splits, hip.stream_handle())
    return out.view(-1)[: splits * m * n].view(splits, m, n)


# ------------------------------------------------------------------ epilogues --
def epilogue_store(part: torch.Tensor, out_dtype: torch.dtype, residual: torch.Tensor | None = None, out=None):
    splits, m, n = part.shape
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=part.device)
    if residual is not None:
        _cuda(residual, "residual")
        _req(residual.numel() == m * n and residual.dtype == out.dtype, "residual must match the output")
    hip.call("cir_epilogue_store", part.data_ptr(), splits, hip.ptr(residual), out.data_ptr(), hip.dtype_code(out.dtype),
             m, n, hip.stream_handle())
    return out


def epilogue_residual_rmsnorm(part: torch.Tensor, residual: torch.Tensor, norm_w: torch.Tensor, eps: float,
                              h_out: torch.Tensor, xn_out: torch.Tensor):
    """h_out = residual + sum(part) (fp32); xn_out = RMSNorm(h_out) * norm_w (GEMM input dtype)."""
    splits, m, n = part.shape
    for t, nm in ((residual, "residual"), (h_out, "h_out"), (xn_out, "xn_out"), (norm_w, "norm_w")):
        _cuda(t, nm)
    _req(residual.dtype == torch.float32 and h_out.dtype == torch.float32, "residual/h_out must be float32", TypeError)
    _req(residual.numel() == m * n and h_out.numel() == m * n and xn_out.numel() == m * n and norm_w.numel() == n,
         "residual_rmsnorm shape mismatch")
    hip.call("cir_epilogue_residual_rmsnorm", part.data_ptr(), splits, residual.data_ptr(), h_out.data_ptr(),
             norm_w.data_ptr(), hip.dtype_code(norm_w.dtype), float(eps), xn_out.data_ptr(),
             hip.dtype_code(xn_out.dtype), m, n, hip.stream_handle())
    return h_out, xn_out


def epilogue_swiglu(part: torch.Tensor, out_dtype: torch.dtype, out=None):
    splits, m, n2 = part.shape
    _req(n2 % 2 == 0, "swiglu partials need gate|up columns")
    inter = n2 // 2
    if out is None:
        out = torch.empty((m, inter), dtype=out_dtype, device=part.device)
    hip.call("cir_epilogue_swiglu", part.data_ptr(), splits, out.data_ptr(), hip.dtype_code(out.dtype), m, inter,
             hip.stream_handle())
    return out


def epilogue_qkv_rope_append(part, inv_freq, positions, page_table, q_out, k_pool, v_pool, *, batch: int, q_len: int,
                             num_heads: int, num_kv_heads: int, head_dim: int) -> torch.Tensor:
    splits, rows, n = part.shape
    _req(rows == batch * q_len and n == (num_heads + 2 * num_kv_heads) * head_dim, "qkv partial shape mismatch")
    _req(positions.dtype == torch.int32 and positions.numel() == batch, "positions must be int32 [batch]")
    _req(page_table.dtype == torch.int32 and page_table.shape[0] == batch, "page_table must be int32 [batch, pages]")
    _req(k_pool.shape[1:] == (num_kv_heads, k_pool.shape[2], head_dim), "pool shape mismatch")
    _req(inv_freq.numel() == head_dim // 2 and inv_freq.dtype == torch.float32, "inv_freq must be float32 [D/2]")
    hip.call("cir_epilogue_qkv_rope_append", part.data_ptr(), splits, inv_freq.data_ptr(), positions.data_ptr(),
             page_table.data_ptr(), page_table.shape[1], q_out.data_ptr(), hip.dtype_code(q_out.dtype),
             k_pool.data_ptr(), v_pool.data_ptr(), hip.dtype_code(k_pool.dtype), batch, q_len, num_heads,
             num_kv_heads, head_dim, k_pool.shape[2], hip.stream_handle())
    return q_out


# ---------------------------------------------------------------- row kernels --
def embedding(ids: torch.Tensor, table: torch.Tensor, out_dtype: torch.dtype, out=None) -> torch.Tensor:
    _cuda(ids, "ids")
    _cuda(table, "table")
    _req(ids.dtype == torch.int64, "ids must be int64", TypeError)
    rows = ids.numel()
    vocab, hidden = table.shape
    if out is None:
        out = torch.empty((rows, hidden), dtype=out_dtype, device=table.device)
    hip.call("cir_embedding", ids.data_ptr(), table.data_ptr(), hip.dtype_code(table.dtype), out.data_ptr(),
             hip.dtype_code(out.dtype), rows, hidden, vocab, hip.stream_handle())
    return out


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, out_dtype: torch.dtype, out=None) -> torch.Tensor:
    _cuda(x, "x")
    _cuda(w, "w")
    hidden = x.shape[-1]
    _req(w.numel() == hidden, "norm weight size mismatch")
    rows = x.numel() // hidden
    if out is None:
        out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    hip.call("cir_rmsnorm", x.data_ptr(), hip.dtype_code(x.dtype), w.data_ptr(), hip.dtype_code(w.dtype),
             out.data_ptr(), hip.dtype_code(out.dtype), rows, hidden, float(eps), hip.stream_handle())
    return out


def add(a: torch.Tensor, b: torch.Tensor, out=None) -> torch.Tensor:
    _cuda(a, "a")
    _cuda(b, "b")
    _req(a.shape == b.shape and a.dtype == b.dtype, "add operands must match")
    out = torch.empty_like(a) if out is None else out
    hip.call("cir_add", a.data_ptr(), b.data_ptr(), out.data_ptr(), hip.dtype_code(a.dtype), a.numel(),
             hip.stream_handle())
    return out


def cast(x: torch.Tensor, dtype: torch.dtype, out=None) -> torch.Tensor:
    _cuda(x, "x")
    out = torch.empty(x.shape, dtype=dtype, device=x.device) if out is None else out
    _req(out.numel() == x.numel(), "cast: size mismatch")
    hip.call("cir_cast", x.data_ptr(), hip.dtype_code(x.dtype), out.data_ptr(), hip.dtype_code(out.dtype), x.numel(),
             hip.stream_handle())
    return out


def argmax(logits: torch.Tensor, out=None) -> torch.Tensor:
    _cuda(logits, "logits")
    _req(logits.dtype == torch.float32 and logits.dim() == 2, "logits must be float32 [rows, vocab]")
    rows, vocab = logits.shape
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    hip.call("cir_argmax", logits.data_ptr(), vocab, out.data_ptr(), rows, vocab, hip.stream_handle())
    return out


def adjust_logits(logits: torch.Tensor, offsets: torch.Tensor | None = None, *, history: torch.Tensor | None = None,
                  history_lens: torch.Tensor | None = None, prompt_lens: torch.Tensor | None = None,
                  drafts: torch.Tensor | None = None, masks: torch.Tensor | None = None,
                  repetition: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                  frequency: torch.Tensor | None = None, bias_ids: torch.Tensor | None = None,
                  bias: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Penalties for repeated tokens, biases and masks on rows of ``logits`` (float32 or float16 ``[rows, vocab]``, any
    row stride).  Sequence b has the rows ``offsets[b] .. offsets[b + 1] - 1`` (int32 ``[B + 1]``; None: a row each),
    tokens ``history[b, : history_lens[b]]`` (int64 ``[B, L]``, int32 ``[B]``; the first ``prompt_lens[b]`` count for
    ``repetition`` only), and, where ``drafts`` (int64 ``[rows]``) and ``masks`` (``draft_tree``) are given, the drafted
    tokens on the row's path (the history ends before them, and before the token that opens the tree, which is one of
    them: what stands in both counts twice).  ``repetition``, ``presence``, ``frequency``: float32 ``[B]``; ``bias_ids`` (int64, -1:
    unused) and ``bias`` (float32) ``[B, K]``; ``allowed``: int32 ``[rows, ceil(vocab / 32)]``, a bit per token.  ``out``
    may be ``logits``.  See ``cir_adjust_logits``."""
    _req(isinstance(logits, torch.Tensor), "logits must be a torch.Tensor", TypeError)
    dev, dt, i32, i64, f32 = logits.get_device(), logits.dtype, torch.int32, torch.int64, torch.float32
    _req(dev >= 0, "logits must be on the GPU")
    shape = logits.shape
    _req(len(shape) == 2 and shape[1] > 0 and (logits.stride(1) == 1 or shape[1] == 1),
         "logits must be [rows, vocab] with contiguous rows")
    rows, vocab = shape
    batch = rows if offsets is None else offsets.numel() - 1
    width = 0 if history is None else history.shape[-1]
    listed = 0 if bias_ids is None else bias_ids.shape[-1]
    words = 0 if masks is None else masks.shape[-1]
    _int32(rows, vocab, batch, width, listed, words)
    for name, t, dtype, want in (
            ("offsets", offsets, i32, (batch + 1,)), ("history", history, i64, (batch, width)),
            ("history_lens", history_lens, i32, (batch,)), ("prompt_lens", prompt_lens, i32, (batch,)),
            ("drafts", drafts, i64, (rows,)), ("masks", masks, i64, (rows, words)),
            ("repetition", repetition, f32, (batch,)), ("presence", presence, f32, (batch,)),
            ("frequency", frequency, f32, (batch,)), ("bias_ids", bias_ids, i64, (batch, listed)),
            ("bias", bias, f32, (batch, listed)), ("allowed", allowed, i32, (rows, (vocab + 31) // 32))):
        if t is not None and not _fits(t, dev, dtype, want):
            _tensors(logits.device, **{name: (t, dtype, want)})
    if (history is None) != (history_lens is None) or (drafts is None) != (masks is None) or (bias is None) != (bias_ids is None):
        _req(False, "history and history_lens, drafts and masks, bias and bias_ids go together")
    _req(prompt_lens is None or history is not None, "prompt_lens needs history")
    _req(drafts is None or offsets is not None, "drafts need offsets")
    ld = logits.stride(0) if rows > 1 else vocab
    if out is None:
        out = torch.empty(shape, dtype=dt, device=logits.device)
        ld_out = vocab
    else:
        _req(isinstance(out, torch.Tensor) and out.device == logits.device and out.shape == shape and out.dtype == dt and
             (out.stride(1) == 1 or vocab == 1), "out must be like logits")
        ld_out = out.stride(0) if rows > 1 else vocab
    ptr = hip.ptr
    _call_on(dev, "cir_adjust_logits", logits.data_ptr(), ld, out.data_ptr(), ld_out, hip.dtype_code(dt), ptr(offsets),
             ptr(history), ptr(history_lens), ptr(prompt_lens), width, ptr(drafts), ptr(masks), words, ptr(repetition),
             ptr(presence), ptr(frequency), ptr(bias_ids), ptr(bias), listed, ptr(allowed), rows, batch, vocab)
    return out


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor | None  # float32 [rows] of the given tokens
    entropy: torch.Tensor          # float32 [rows], in nats
    top_ids: torch.Tensor          # int64 [rows, top_k], most likely first
    top_logprobs: torch.Tensor     # float32 [rows, top_k]


def token_logprobs_workspace(rows: int, vocab: int, top_k: int, device) -> torch.Tensor:
    return torch.empty(max(hip.size_call("cir_token_logprobs_workspace_bytes", rows, vocab, top_k), 8),
                       dtype=torch.uint8, device=device)


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor | None, top_k: int = 0, *,
                   workspace: torch.Tensor | None = None) -> TokenLogprobs:
    """Log probabilities of ``ids`` (int64 ``[rows]``; an id outside the vocabulary gives NaN), entropy and the ``top_k``
    (0..64) most likely tokens of each row of ``logits`` (float32 or float16 ``[rows, vocab]``, any row stride) in one
    pass, for fewer than 2**24 rows.  Ties go to the lowest id, NaN counts as the largest logit; see
    ``cir_token_logprobs``."""
    _req(isinstance(logits, torch.Tensor), "logits must be a torch.Tensor", TypeError)
    dev = logits.get_device()
    _req(dev >= 0, "logits must be on the GPU")
    _req(logits.dim() == 2 and logits.shape[1] > 0 and (logits.stride(1) == 1 or logits.shape[1] == 1),
         "logits must be [rows, vocab] with contiguous rows")
    rows, vocab = logits.shape
    _int32(rows, vocab)
    ld = logits.stride(0) if rows > 1 else vocab
    _req(ld >= vocab, "logits rows overlap")
    if not (0 <= top_k <= 64 and top_k <= vocab):
        _req(False, f"top_k must be 0..64 and at most the vocabulary (got {top_k})")
    code = hip.dtype_code(logits.dtype)
    if ids is not None and not _fits(ids, dev, torch.int64, (rows,)):
        _tensors(logits.device, ids=(ids, torch.int64, (rows,)))
    # one allocation for what is float32
    n = 0 if ids is None else rows
    lp, entropy, top_lp = torch.empty(n + rows + rows * top_k, dtype=torch.float32,
                                      device=logits.device).split_with_sizes((n, rows, rows * top_k))
    res = TokenLogprobs(None if ids is None else lp, entropy,
                        torch.empty((rows, top_k), dtype=torch.int64, device=logits.device), top_lp.view(rows, top_k))
    if workspace is not None:
        _check_workspace(workspace, dev)
    elif hip.size_call("cir_token_logprobs_workspace_bytes", rows, vocab, top_k):
        workspace = token_logprobs_workspace(rows, vocab, top_k, logits.device)
    ws, ws_bytes = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.nbytes)
    _call_on(dev, "cir_token_logprobs", logits.data_ptr(), code, ld, hip.ptr(ids), rows, vocab, top_k, lp.data_ptr(),
             entropy.data_ptr(), res.top_ids.data_ptr(), top_lp.data_ptr(), ws, ws_bytes)
    return res


def stream_read(buf: torch.Tensor, workgroups: int, threads: int, layout: int, out: torch.Tensor,
                side: torch.Tensor | None = None, side_ratio: int = 0) -> None:
    """Read every byte of ``buf`` (``cir_stream_read``; read-bandwidth calibration, not on the decode path), with
    ``side_ratio`` 16-byte reads of the L2-resident ``side`` per 8 of ``buf``."""
    _cuda(buf, "buf")
    _cuda(out, "out")
    sp, sb = 0, 0
    if side is not None:
        _cuda(side, "side")
        sp, sb = side.data_ptr(), side.numel() * side.element_size()
    hip.call("cir_stream_read", buf.data_ptr(), buf.numel() * buf.element_size(), int(workgroups), int(threads),
             int(layout), sp, sb, int(side_ratio), out.data_ptr(), hip.stream_handle())
