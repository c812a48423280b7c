"""torch-tensor front ends of the kernel-level C ABI (include/fasttalk_b200.h).  PyTorch only
supplies device memory and the stream; all arithmetic happens in the CUDA library."""
from __future__ import annotations

from typing import Optional

import torch

from . import native as N

KV_TILE = 64


def _chk_bf16(t, name):
    assert t.is_cuda and t.dtype == torch.bfloat16 and t.is_contiguous(), f"{name}: need contiguous CUDA bf16"


def split_hi_lo(x: torch.Tensor):
    """fp32 -> (bf16 hi, bf16 lo) planes with hi + lo ~= x to ~16 mantissa bits."""
    hi = x.to(torch.bfloat16)
    lo = (x.float() - hi.float()).to(torch.bfloat16)
    return hi.contiguous(), lo.contiguous()


def gemm_bf16(w: torch.Tensor, x: torch.Tensor, x_lo: Optional[torch.Tensor] = None, n_splits: int = 0,
              mode: str = "partials"):
    """Y[t, n] = sum_k (X + Xlo)[t, k] W[n, k].
    mode "partials": fp32 [S, T, n_out]; "bf16": (hi, lo) bf16 [T, n_out];
    "swiglu": w rows interleaved gate|up per 64 -> (hi, lo) bf16 [T, n_out/2]."""
    _chk_bf16(w, "w"); _chk_bf16(x, "x")
    if x_lo is not None:
        _chk_bf16(x_lo, "x_lo")
    n_out, K = w.shape
    T = x.shape[0]
    assert x.shape[1] == K
    lib = N.load()
    st = N.cur_stream()
    if mode == "partials":
        if n_splits <= 0:
            n_splits = lib.ft_gemm_pick_parts(n_out, T, K, int(x_lo is not None))
        out = torch.empty(n_splits, T, n_out, device=x.device, dtype=torch.float32)
        N.check(lib.ft_gemm_bf16(N.ptr(w), N.ptr(x), N.ptr(x_lo), N.ptr(out), 0, n_out, T, K, n_splits, 0, st),
                "ft_gemm_bf16")
        return out
    width = n_out if mode == "bf16" else n_out // 2
    out = torch.empty(T, width, device=x.device, dtype=torch.bfloat16)
    out_lo = torch.empty_like(out)
    N.check(lib.ft_gemm_bf16(N.ptr(w), N.ptr(x), N.ptr(x_lo), N.ptr(out), N.ptr(out_lo), n_out, T, K, 1,
                             1 if mode == "bf16" else 2, st), "ft_gemm_bf16")
    return out, out_lo


def gemm_fused(w: torch.Tensor, x: torch.Tensor, x_lo: torch.Tensor, mode: int, n_splits: int = 0, **f) -> None:
    """ft_gemm_fused with an ft_gemm_epilogue built from keyword tensors / scalars (see
    include/fasttalk_b200.h).  Outputs are whatever tensors the caller put in the epilogue."""
    import ctypes as C
    if f.get("x_planes") == 3:       # the fp16 single-plane form of the large prefill projections: fp16 weights, x_lo = None
        assert x_lo is None and all(t.is_cuda and t.dtype == torch.float16 and t.is_contiguous() for t in (w, x)), \
            "x_planes = 3: need contiguous CUDA fp16 w and x, x_lo = None"
    else:
        _chk_bf16(w, "w"); _chk_bf16(x, "x"); _chk_bf16(x_lo, "x_lo")
    n_out, K = w.shape
    T = x.shape[0]
    ep = N.GemmEpilogue()
    ep.mode = mode
    lib = N.load()
    if mode in (N.EPI_RESID, N.EPI_QKV_ROPE) and "scratch" not in f:
        # split-K work buffers: slabs for the partial tiles + self re-arming arrival counters
        f = dict(f)
        f["scratch"] = torch.empty(max(1, lib.ft_gemm_scratch_bytes(n_out, T, K, n_splits) // 4), device=x.device,
                                   dtype=torch.float32)
        f["sync"] = torch.zeros(2 * (n_out // 128) * ((T + 15) // 16), device=x.device, dtype=torch.int32)
    for name, _ in N.GemmEpilogue._fields_:
        if name == "mode" or name not in f:
            continue
        v = f[name]
        setattr(ep, name, v.data_ptr() if isinstance(v, torch.Tensor) else v)
    N.check(N.load().ft_gemm_fused(N.ptr(w), N.ptr(x), N.ptr(x_lo), n_out, T, K, n_splits, C.byref(ep),
                                   N.cur_stream()), "ft_gemm_fused")


def embed_planes(tokens: torch.Tensor, table: torch.Tensor, gamma: torch.Tensor, ssq_parts: int):
    """resid = table[tokens] (fp32); planes = hi/lo(resid * gamma); ssq [parts, T]."""
    T, h = tokens.numel(), table.shape[1]
    resid = torch.empty(T, h, device=table.device, dtype=torch.float32)
    hi = torch.empty(T, h, device=table.device, dtype=torch.bfloat16)
    lo = torch.empty_like(hi)
    ssq = torch.empty(ssq_parts, T, device=table.device, dtype=torch.float32)
    N.check(N.load().ft_embed_planes(N.ptr(tokens), N.ptr(table), N.ptr(gamma), N.ptr(resid), N.ptr(hi), N.ptr(lo),
                                     N.ptr(ssq), ssq_parts, T, T, h, N.cur_stream()), "ft_embed_planes")
    return resid, hi, lo, ssq


def gather_planes(x: torch.Tensor, x_lo: torch.Tensor, ssq: torch.Tensor, row_idx: torch.Tensor):
    n, h = row_idx.numel(), x.shape[1]
    hi = torch.empty(n, h, device=x.device, dtype=torch.bfloat16)
    lo = torch.empty_like(hi)
    so = torch.empty(ssq.shape[0], n, device=x.device, dtype=torch.float32)
    N.check(N.load().ft_gather_planes(N.ptr(x), N.ptr(x_lo), N.ptr(ssq), ssq.shape[0], ssq.stride(0), N.ptr(row_idx),
                                      n, h, N.ptr(hi), N.ptr(lo), N.ptr(so), n, N.cur_stream()), "ft_gather_planes")
    return hi, lo, so


def add_rmsnorm(resid: torch.Tensor, norm_w: torch.Tensor, eps: float, partials: Optional[torch.Tensor] = None,
                embed_tokens: Optional[torch.Tensor] = None, embed_table: Optional[torch.Tensor] = None,
                row_idx: Optional[torch.Tensor] = None):
    """In-place residual update + RMSNorm; returns the bf16 (hi, lo) planes [n_rows, h]."""
    assert resid.dtype == torch.float32 and resid.is_contiguous()
    h = resid.shape[1]
    T = row_idx.numel() if row_idx is not None else resid.shape[0]
    xn = torch.empty(T, h, device=resid.device, dtype=torch.bfloat16)
    xn_lo = torch.empty_like(xn)
    ns, stride = 0, 0
    if partials is not None:
        assert partials.dtype == torch.float32 and partials.is_contiguous()
        ns, stride = partials.shape[0], partials.stride(0)
    N.check(N.load().ft_add_rmsnorm(N.ptr(resid), N.ptr(partials), ns, stride, N.ptr(embed_tokens),
                                    N.ptr(embed_table), N.ptr(norm_w), N.ptr(xn), N.ptr(xn_lo), N.ptr(row_idx),
                                    T, h, eps, N.cur_stream()), "ft_add_rmsnorm")
    return xn, xn_lo


def kv_cache_alloc(num_pages: int, nkv: int, d: int, device) -> torch.Tensor:
    """One layer of paged KV cache: [page][kv_head][K|V][64][d] fp16 (swizzled rows)."""
    return torch.zeros(num_pages, nkv, 2, KV_TILE, d, device=device, dtype=torch.float16)


def rope_kv_append(qkv_partials: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                   seq_rows: torch.Tensor, page_table: torch.Tensor, kv_layer: torch.Tensor,
                   nq: int, nkv: int, d: int) -> torch.Tensor:
    S, T, _ = qkv_partials.shape
    q = torch.empty(T, nq, d, device=qkv_partials.device, dtype=torch.float16)
    N.check(N.load().ft_rope_kv_append(N.ptr(qkv_partials), S, qkv_partials.stride(0), N.ptr(cos), N.ptr(sin),
                                       N.ptr(positions), N.ptr(seq_rows), N.ptr(page_table),
                                       page_table.shape[1], N.ptr(q), N.ptr(kv_layer), T, nq, nkv, d,
                                       N.cur_stream()), "ft_rope_kv_append")
    return q


def silu_mul(gu_partials: torch.Tensor):
    S, T, f2 = gu_partials.shape
    act = torch.empty(T, f2 // 2, device=gu_partials.device, dtype=torch.bfloat16)
    act_lo = torch.empty_like(act)
    N.check(N.load().ft_silu_mul(N.ptr(gu_partials), S, gu_partials.stride(0), N.ptr(act), N.ptr(act_lo), T,
                                 f2 // 2, N.cur_stream()), "ft_silu_mul")
    return act, act_lo


def attn_decode(q: torch.Tensor, kv_layer: torch.Tensor, page_table: torch.Tensor, ctx_lens: torch.Tensor,
                n_ctas: int = 0):
    """q fp16 [B, nq, d], fp16 KV cache -> bf16 (hi, lo) planes [B, nq*d]."""
    assert q.dtype == torch.float16 and kv_layer.dtype == torch.float16
    B, nq, d = q.shape
    nkv = kv_layer.shape[1]
    lib = N.load()
    if n_ctas <= 0:
        n_ctas = N.check(lib.ft_attn_decode_default_ctas(d), "ft_attn_decode_default_ctas")
    scratch = torch.empty(lib.ft_attn_decode_scratch_bytes(B, nkv, nq // nkv, d, n_ctas) // 4,
                          device=q.device, dtype=torch.float32)
    tile_prefix = torch.empty(B + 1, device=q.device, dtype=torch.int32)
    out = torch.empty(B, nq * d, device=q.device, dtype=torch.bfloat16)
    out_lo = torch.empty_like(out)
    N.check(lib.ft_attn_decode(N.ptr(q), N.ptr(kv_layer), N.ptr(page_table), page_table.shape[1],
                               N.ptr(ctx_lens), N.ptr(tile_prefix), N.ptr(out), N.ptr(out_lo), N.ptr(scratch), B,
                               nq, nkv, d, n_ctas, N.cur_stream()), "ft_attn_decode")
    return out, out_lo


def attn_decode_noalloc(q: torch.Tensor, kv_layer: torch.Tensor, page_table: torch.Tensor, ctx_lens: torch.Tensor,
                        out: torch.Tensor, out_lo: torch.Tensor, n_ctas: int = 0) -> None:
    """Decode attention for callers that may not allocate device memory while serving (fixed
    start-up memory budget, real-time audio thread): the library's built-in work area replaces
    the scratch buffers attn_decode() allocates, and the caller supplies `out` / `out_lo`
    (bf16 [B, nq*d]) itself, so this call allocates nothing anywhere.  Calls on one GPU share
    that work area: do not overlap them.  Raises NativeError beyond B*nkv = 1024 / n_ctas = 512."""
    B, nq, d = q.shape
    nkv = kv_layer.shape[1]
    N.check(N.load().ft_attn_decode_noalloc(N.ptr(q), N.ptr(kv_layer), N.ptr(page_table), page_table.shape[1],
                                            N.ptr(ctx_lens), N.ptr(out), N.ptr(out_lo), B, nq, nkv, d, n_ctas,
                                            N.cur_stream()), "ft_attn_decode_noalloc")


def attn_prefill(q: torch.Tensor, kv_layer: torch.Tensor, page_table: torch.Tensor, req_q_start, req_slot,
                 req_pos0, tensor_cores: bool = True):
    """q fp16 [T, nq, d]; request r owns rows req_q_start[r]:req_q_start[r+1].  Returns (hi, lo)."""
    assert q.dtype == torch.float16 and kv_layer.dtype == torch.float16
    T, nq, d = q.shape
    nkv = kv_layer.shape[1]
    dev = q.device
    tile_req, tile_q0 = [], []
    for r in range(len(req_slot)):
        for q0 in range(0, req_q_start[r + 1] - req_q_start[r], 64):
            tile_req.append(r); tile_q0.append(q0)
    # The lists go up in one copy that the host does not wait for (five waiting ones cost 60 us of GPU time between calls).  While a
    # stream is captured the copy is an ordinary one, which capture refuses: a replay would read memory that is no longer this call's.
    i32 = lambda v: torch.tensor(v, device="cpu", dtype=torch.int32).reshape(-1)
    n = len(tile_req)
    parts = [i32(v) for v in (req_q_start, req_slot, req_pos0, tile_req + tile_q0)]
    assert parts[2].numel() >= len(req_slot), "req_pos0: a position for every request"
    rows = T if tensor_cores else 0
    lib = N.load()
    tiles = N.ptr(parts[3])
    few = N.check(lib.ft_attn_prefill_order_tiles(N.ptr(parts[0]), N.ptr(parts[2]), tiles, tiles + 4 * n, n, nq, nkv, d, rows), "ft_attn_prefill_order_tiles")
    lists = torch.cat(parts)
    waits = dev.index != torch.cuda.current_device() or torch.cuda.is_current_stream_capturing()
    lists = lists.to(dev) if waits else lists.pin_memory().to(dev, non_blocking=True)
    t_qs, t_slot, t_pos0, t_treq, t_tq0 = lists.split([p.numel() for p in parts[:3]] + [n, n])
    # rows that no request owns are zeros
    starts = parts[0].tolist()[:len(req_slot) + 1]
    owned = bool(starts) and starts[0] == 0 and starts[-1] == T and all(x <= y for x, y in zip(starts, starts[1:]))
    out = (torch.empty if owned else torch.zeros)(T, nq * d, device=dev, dtype=torch.bfloat16)
    out_lo = torch.empty_like(out) if owned else torch.zeros_like(out)
    N.check(lib.ft_attn_prefill_ordered(N.ptr(q), N.ptr(kv_layer), N.ptr(page_table), page_table.shape[1],
                                        N.ptr(t_qs), N.ptr(t_slot), N.ptr(t_pos0), N.ptr(t_treq), N.ptr(t_tq0),
                                        n, N.ptr(out), N.ptr(out_lo), nq, nkv, d, rows, few, N.cur_stream()),
            "ft_attn_prefill")
    return out, out_lo


def sample(logits: torch.Tensor, temperature=None, top_k=None, top_p=None, seeds=None) -> torch.Tensor:
    B, V = logits.shape
    assert logits.dtype == torch.float32 and logits.is_contiguous()
    out = torch.empty(B, device=logits.device, dtype=torch.int32)
    N.check(N.load().ft_sample(N.ptr(logits), B, V, N.ptr(temperature), N.ptr(top_k), N.ptr(top_p),
                               N.ptr(seeds), N.ptr(out), N.cur_stream()), "ft_sample")
    return out


# ---- the 8-bit KV cache: the four steps above over a cache of half the bytes
# One layer is uint8 [pages][kv heads][128 d + 32]: per page and head the key codes, the value codes and eight fp32 scales, one for each block of 16 tokens of
# keys and of values (csrc/kv8.cuh has the order of the codes; kv8_codes / kv8_records below).  A code c stands for (c - 128) * scale.
KV8_BLOCK = 16


def _refuse(what: str, why: str) -> None:
    raise N.NativeError(f"{what}: {why}")


# The checks below run ahead of every call: a step of single tokens takes a few microseconds on the GPU, so they ask tensors for numbers, not for objects.
def _kv8_layer(layer: torch.Tensor, d: int, what: str):
    """(device, pages, kv heads) of a layer; all tensors of a call have to be on its device."""
    index = layer.get_device()
    if index < 0 or layer.dtype is not torch.uint8 or layer.dim() != 3 or not layer.is_contiguous():
        _refuse(what, "the cache is contiguous CUDA uint8 [pages, nkv, record]")
    pages, nkv, record = layer.shape
    if record != 128 * d + 32:
        _refuse(what, "the cache's records are not those of this head_dim")
    return index, pages, nkv


def _kv8_ints(t, index: int, what: str, n: int, name: str) -> torch.Tensor:
    """int32 on the device, n of them (n < 0: any number); a list goes up in a copy that the host waits for."""
    if not isinstance(t, torch.Tensor):
        t = torch.tensor(t, dtype=torch.int32, device=f"cuda:{index}").reshape(-1)
    if t.dtype is not torch.int32 or t.get_device() != index or not t.is_contiguous():
        _refuse(what, f"{name} is contiguous int32 on the cache's device")
    if n >= 0 and t.numel() != n:
        _refuse(what, f"{name} has {n} numbers here, not {t.numel()}")
    return t


def _kv8_table(t: torch.Tensor, index: int, what: str):
    if t.dtype is not torch.int32 or t.get_device() != index or t.dim() != 2 or not t.is_contiguous():
        _refuse(what, "page_table is contiguous int32 [sequences, pages] on the cache's device")
    return t.shape


def _kv8_requests(req_start, req_slot, req_pos0, index: int, what: str):
    req_slot = _kv8_ints(req_slot, index, what, -1, "req_slot")
    n = req_slot.numel()
    return _kv8_ints(req_start, index, what, n + 1, "req_start"), req_slot, _kv8_ints(req_pos0, index, what, n, "req_pos0"), n


def _kv8_call(index: int, name: str, *args) -> None:
    """A library call on the device's current stream, whichever device is the current one."""
    fn, stream = getattr(N.load(), name), torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc < 0:
        N.check(rc, name)


_kv8_sizes = {}


def _kv8_sms(index: int) -> int:
    n = _kv8_sizes.get(index)
    if n is None:
        n = _kv8_sizes[index] = torch.cuda.get_device_properties(index).multi_processor_count
    return n


def _kv8_scratch(index: int, name: str, d: int) -> torch.Tensor:
    n = _kv8_sizes.get((index, name, d))
    if n is None:
        with torch.cuda.device(index):
            n = _kv8_sizes[index, name, d] = N.check(getattr(N.load(), name)(d), name)
    return torch.empty(n, device=index, dtype=torch.uint8)


def kv8_cache_alloc(num_pages: int, nkv: int, d: int, device) -> torch.Tensor:
    """One layer of 8-bit KV cache, all zeros."""
    if d not in (64, 128):
        _refuse("kv8_cache_alloc", "head_dim 64 or 128")
    return torch.zeros(num_pages, nkv, 128 * d + 32, device=device, dtype=torch.uint8)


def rope_kv8_append(qkv_partials: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, seq_rows: torch.Tensor,
                    page_table: torch.Tensor, kv8_layer: torch.Tensor, nq: int, nkv: int, d: int) -> torch.Tensor:
    """rope_kv_append into the 8-bit cache -> q fp16 [T, nq, d].  Tokens of one sequence stand side by side in `positions` / `seq_rows`, without gaps.  A block
    whose scale is too small for a new token is rescaled, the tokens before it in the block with it; a block that is entered at its first token starts anew.
    Tokens without a place (a position outside the tables, a page outside the cache) are not written."""
    what = "rope_kv8_append"
    index, pages, heads = _kv8_layer(kv8_layer, d, what)
    width = (nq + 2 * nkv) * d
    if heads != nkv:
        _refuse(what, "the cache has another number of heads")
    if qkv_partials.dim() != 3 or qkv_partials.dtype is not torch.float32 or qkv_partials.get_device() != index or qkv_partials.shape[2] != width:
        _refuse(what, "qkv_partials is fp32 [S, T, (nq + 2 nkv) d] on the cache's device")
    S, T, _ = qkv_partials.shape
    part, row, one = qkv_partials.stride()
    if one != 1 or (row != width and T > 1):
        _refuse(what, "the rows of qkv_partials lie one behind the other")
    if (cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or cos.get_device() != index or sin.get_device() != index or cos.dim() != 2
            or cos.shape != sin.shape or cos.shape[1] * 2 != d or not cos.is_contiguous() or not sin.is_contiguous()):
        _refuse(what, "cos and sin are contiguous fp32 [positions, d / 2] on the cache's device")
    positions, seq_rows = _kv8_ints(positions, index, what, T, "positions"), _kv8_ints(seq_rows, index, what, T, "seq_rows")
    rows, most = _kv8_table(page_table, index, what)
    q = torch.empty(T, nq, d, device=index, dtype=torch.float16)
    _kv8_call(index, "ft_rope_kv8_append", qkv_partials.data_ptr(), S, part, cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(),
              seq_rows.data_ptr(), page_table.data_ptr(), rows, most, q.data_ptr(), kv8_layer.data_ptr(), pages, T, nq, nkv, d)
    return q


def kv8_read(kv8_layer: torch.Tensor, page_table: torch.Tensor, req_start, req_slot, req_pos0, rows: int, d: int):
    """Keys and values back as fp16 [rows, nkv, d] each: request r gets rows req_start[r] .. req_start[r + 1] - 1, from position req_pos0[r] of page-table row
    req_slot[r] on.  Rows that no request owns, and rows without a page, are zeros.  The lists are int32 tensors on the device, or anything a tensor is made of."""
    what = "kv8_read"
    index, pages, nkv = _kv8_layer(kv8_layer, d, what)
    table_rows, most = _kv8_table(page_table, index, what)
    req_start, req_slot, req_pos0, n = _kv8_requests(req_start, req_slot, req_pos0, index, what)
    if rows < 0:
        _refuse(what, "a number of rows")
    k = torch.empty(rows, nkv, d, device=index, dtype=torch.float16)
    v = torch.empty_like(k)
    _kv8_call(index, "ft_kv8_read", kv8_layer.data_ptr(), pages, page_table.data_ptr(), table_rows, most, req_start.data_ptr(), req_slot.data_ptr(),
              req_pos0.data_ptr(), n, rows, k.data_ptr(), v.data_ptr(), nkv, d)
    return k, v


def _kv8_query(q: torch.Tensor, kv8_layer: torch.Tensor, planes: int, what: str):
    if q.dim() != 3 or q.dtype is not torch.float16 or not q.is_contiguous():
        _refuse(what, "q is contiguous fp16 [rows, nq, d]")
    rows, nq, d = q.shape
    index, pages, nkv = _kv8_layer(kv8_layer, d, what)
    if q.get_device() != index:
        _refuse(what, "q is on another device than the cache")
    if planes != 1 and planes != 2:
        _refuse(what, "one plane or two")
    out = torch.empty(rows, nq * d, device=index, dtype=torch.bfloat16)
    return index, pages, nkv, rows, nq, d, out, torch.empty_like(out) if planes == 2 else None


def attn_decode_kv8(q: torch.Tensor, kv8_layer: torch.Tensor, page_table: torch.Tensor, ctx_lens: torch.Tensor, planes: int = 2):
    """attn_decode over the 8-bit cache: q fp16 [B, nq, d], up to eight query heads a key head -> bf16 (hi, lo) planes [B, nq * d], lo None with planes = 1.  A
    sequence without keys gives zeros; keys on pages outside the cache are hidden."""
    what = "attn_decode_kv8"
    index, pages, nkv, B, nq, d, out, lo = _kv8_query(q, kv8_layer, planes, what)
    ctx_lens = _kv8_ints(ctx_lens, index, what, B, "ctx_lens")
    rows, most = _kv8_table(page_table, index, what)
    if rows < B:
        _refuse(what, "a page-table row for every query")
    # the library needs none for a few sequences whose page tables are short
    scratch = _kv8_scratch(index, "ft_attn_decode_kv8_scratch_bytes", d) if most > 16 or B * nkv > 2 * _kv8_sms(index) else None
    _kv8_call(index, "ft_attn_decode_kv8", q.data_ptr(), kv8_layer.data_ptr(), pages, page_table.data_ptr(), most, ctx_lens.data_ptr(), out.data_ptr(),
              0 if lo is None else lo.data_ptr(), 0 if scratch is None else scratch.data_ptr(), B, nq, nkv, d)
    return out, lo


def attn_prefill_kv8(q: torch.Tensor, kv8_layer: torch.Tensor, page_table: torch.Tensor, req_q_start, req_slot, req_pos0, planes: int = 2):
    """attn_prefill over the 8-bit cache, up to eight query heads a key head.  The lists are int32 tensors on the device (then nothing goes up, and the call can be
    captured) or anything a tensor is made of.  Rows that no request owns are zeros; keys on pages outside the cache are hidden.  -> (hi, lo), lo None with planes = 1."""
    what = "attn_prefill_kv8"
    index, pages, nkv, T, nq, d, out, lo = _kv8_query(q, kv8_layer, planes, what)
    rows, most = _kv8_table(page_table, index, what)
    req_q_start, req_slot, req_pos0, n = _kv8_requests(req_q_start, req_slot, req_pos0, index, what)
    scratch = _kv8_scratch(index, "ft_attn_prefill_kv8_scratch_bytes", d)
    _kv8_call(index, "ft_attn_prefill_kv8", q.data_ptr(), kv8_layer.data_ptr(), pages, page_table.data_ptr(), rows, most, req_q_start.data_ptr(),
              req_slot.data_ptr(), req_pos0.data_ptr(), n, T, out.data_ptr(), 0 if lo is None else lo.data_ptr(), scratch.data_ptr(), nq, nkv, d)
    return out, lo


def kv8_check(device=None) -> None:
    """Waits for the device (the current one by default) and raises if a kernel of this cache has ever given up on a wait there: rows of some call since the library
    was loaded mean nothing.  No call asks by itself, since that would make the host wait."""
    with torch.cuda.device(device):
        if N.check(N.load().ft_kv8_waits(), "ft_kv8_waits"):
            raise N.NativeError("8-bit KV cache: a wait inside a kernel ran out; outputs of this process are not to be trusted")


def _kv8_offsets(d: int, device) -> torch.Tensor:
    """Where the code of (keys 0 | values 1, token, dim) lies in a record."""
    t, i = torch.arange(KV_TILE, device=device)[:, None], torch.arange(d, device=device)[None, :]
    piece = (i >> 6) * (KV_TILE * 64)
    return torch.stack([piece + t * 64 + (i & 63), KV_TILE * d + piece + (t ^ (t >> 1 & 1)) * 64 + ((i & 63) ^ (t & 4) * 8)])


def kv8_codes(records: torch.Tensor, d: int):
    """records [..., 128 d + 32] as stored -> codes uint8 [..., 2, 64, d], scales fp32 [..., 2, 4]."""
    at = _kv8_offsets(d, records.device)
    scales = records[..., 2 * KV_TILE * d:].contiguous().view(torch.float32)
    return records[..., at.reshape(-1)].reshape(records.shape[:-1] + at.shape), scales.reshape(records.shape[:-1] + (2, KV_TILE // KV8_BLOCK))


def kv8_records(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """inverse of kv8_codes."""
    d, lead = codes.shape[-1], codes.shape[:-3]
    body = torch.empty(lead + (2 * KV_TILE * d,), device=codes.device, dtype=torch.uint8)
    body[..., _kv8_offsets(d, codes.device).reshape(-1)] = codes.reshape(body.shape)
    return torch.cat([body, scales.to(torch.float32).contiguous().reshape(lead + (-1,)).view(torch.uint8)], -1)


# ---- KV cache (un)swizzle helpers for tests: logical [tokens, d] <-> stored slab
# A stored slab is d / 64 sub-slabs of [64 tokens][64 dims]; inside a sub-slab the eight 16-byte chunks of a row are
# XOR-swizzled with the row index (csrc/common.cuh: kv_swizzled_chunk).  The XOR is an involution.
def _kv_perm(x: torch.Tensor) -> torch.Tensor:
    h, rows = x.shape[0], x.shape[1]
    r = torch.arange(rows, device=x.device)[None, :, None]
    c = torch.arange(8, device=x.device)[None, None, :]
    src = (c ^ (r & 7)).expand(h, rows, 8)
    return torch.gather(x, 2, src[..., None].expand(h, rows, 8, 8))


def kv_slab_logical(slab: torch.Tensor) -> torch.Tensor:
    """slab [64, d] as stored (memory order [d/64][64][64]) -> logical [64, d]."""
    rows, d = slab.shape
    x = slab.reshape(d // 64, rows, 8, 8)
    return _kv_perm(x).permute(1, 0, 2, 3).reshape(rows, d)


def kv_slab_store(logical: torch.Tensor) -> torch.Tensor:
    """inverse of kv_slab_logical: logical [64, d] -> the [64, d]-shaped view of the stored bytes."""
    rows, d = logical.shape
    x = logical.reshape(rows, d // 64, 8, 8).permute(1, 0, 2, 3).contiguous()
    return _kv_perm(x).reshape(rows, d)
