"""torch-tensor front end of the libmsgl C ABI (device memory and streams come from torch).

Each function checks shapes / dtypes, then calls the matching ``msgl_*`` entry point on the
current torch stream. No function here computes anything itself.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import check, lib

BF16, F32 = 1, 0
_DT = {torch.bfloat16: BF16, torch.float32: F32}
_SECTIONS = C.c_int * 3


def _s():
    """The current stream's handle. The raw lookup costs 0.2 us; torch.cuda.current_stream() builds
    a Stream object (3.3 us)."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _p(t):
    return None if t is None else t.data_ptr()


def _c(t, dtype=None):
    assert t.is_cuda and t.is_contiguous(), "expected a contiguous CUDA tensor"
    if dtype is not None:
        assert t.dtype == dtype, f"expected {dtype}, got {t.dtype}"
    return t


def _on(dtype, *tensors):
    """Contiguous tensors of one dtype on the current device (whose stream the call uses)."""
    dev = torch._C._cuda_getDevice()
    for t in tensors:
        if t.get_device() != dev or t.dtype != dtype or not t.is_contiguous():
            raise ValueError(f"expected a contiguous {dtype} tensor on cuda:{dev}, got {t.dtype} "
                             f"{tuple(t.shape)} with strides {t.stride()} on {t.device}")


# ------------------------------------------------------------------ reference launchers
def rmsnorm(x, w, eps):
    _c(x), _c(w, x.dtype)
    out = torch.empty_like(x)
    H = w.numel()
    check(lib().msgl_launch_rmsnorm(_p(x), _p(w), _p(out), x.numel() // H, H, eps, _DT[x.dtype], _s()))
    return out


def rope_(q, k, positions, cos_sin, num_q_heads, num_kv_heads, head_dim):
    """In-place rotate-half RoPE on q [T, Hq*D] and k [T, Hkv*D] (k may be None)."""
    _c(q), _c(positions, torch.int32), _c(cos_sin, torch.float32)
    check(lib().msgl_launch_rope(_p(q), _p(k), _p(positions), _p(cos_sin), positions.numel(),
                                 num_q_heads, num_kv_heads, head_dim, _DT[q.dtype], _s()))


def index_gather(table, ids):
    _c(table), _c(ids, torch.int32)
    out = torch.empty(ids.numel(), table.shape[1], dtype=table.dtype, device=table.device)
    check(lib().msgl_launch_index_gather(_p(table), _p(ids), _p(out), table.shape[1], ids.numel(),
                                         table.shape[0], _DT[table.dtype], _s()))
    return out


def store_kv_page(k, v, k_cache, v_cache, page_table, page_size, num_heads, head_dim):
    _c(k), _c(v), _c(k_cache), _c(v_cache), _c(page_table, torch.int32)
    T = k.numel() // (num_heads * head_dim)
    check(lib().msgl_launch_store_kv_page(_p(k), _p(v), _p(k_cache), _p(v_cache), _p(page_table),
                                          page_size, num_heads, head_dim, T, _DT[k.dtype], _s()))


# ------------------------------------------------------------------ fused ops
def add_rmsnorm_(x, residual, w, eps, first=False):
    """In place: residual += x (or = x when first); x = rmsnorm(residual) * w."""
    _c(x, torch.bfloat16), _c(residual, torch.float32), _c(w, torch.bfloat16)
    H = w.numel()
    check(lib().msgl_add_rmsnorm(_p(x), _p(residual), _p(w), x.numel() // H, H, eps, int(first), _s()))


def add_partials_rmsnorm_(parts, x, residual, w, eps):
    """residual += sum_p parts[p] (fp32 split-K partials [P, T, H], added in p order);
    x = rmsnorm(residual) * w (x written in place)."""
    _c(parts, torch.float32), _c(x, torch.bfloat16), _c(residual, torch.float32), _c(w, torch.bfloat16)
    H = w.numel()
    T = x.numel() // H
    check(lib().msgl_add_partials_rmsnorm(_p(parts), parts.numel() // (T * H), _p(x), _p(residual),
                                          _p(w), T, H, eps, _s()))


def embed_rmsnorm(embed, ids, w, eps):
    _c(embed, torch.bfloat16), _c(ids, torch.int32), _c(w, torch.bfloat16)
    V, H = embed.shape
    x = torch.empty(ids.numel(), H, dtype=torch.bfloat16, device=embed.device)
    r = torch.empty(ids.numel(), H, dtype=torch.float32, device=embed.device)
    check(lib().msgl_embed_rmsnorm(_p(embed), _p(ids), ids.numel(), V, H, _p(w), eps, _p(x), _p(r), _s()))
    return x, r


def qknorm_rope_store_kv(qkv, k_pool, v_pool, positions, slot_mapping, cos_sin, q_norm, k_norm,
                         num_q_heads, num_kv_heads, eps, head_dim=128):
    _c(qkv, torch.bfloat16), _c(k_pool, torch.bfloat16), _c(v_pool, torch.bfloat16)
    _c(positions, torch.int32), _c(slot_mapping, torch.int32), _c(cos_sin, torch.float32)
    T = positions.numel()
    q = torch.empty(T, num_q_heads, head_dim, dtype=torch.bfloat16, device=qkv.device)
    num_slots = k_pool.numel() // (num_kv_heads * head_dim)
    check(lib().msgl_qknorm_rope_store_kv(_p(qkv), _p(q), _p(k_pool), _p(v_pool), num_slots,
                                          _p(positions), _p(slot_mapping), _p(cos_sin), _p(q_norm),
                                          _p(k_norm), T, num_q_heads, num_kv_heads, head_dim, eps, _s()))
    return q


def qknorm_rope_store_kv_partials(parts, k_pool, v_pool, positions, slot_mapping, cos_sin, q_norm,
                                  k_norm, num_q_heads, num_kv_heads, eps, head_dim=128):
    """As qknorm_rope_store_kv with the QKV rows the sum of fp32 partials [P, T, (Hq+2Hkv) D]."""
    _c(parts, torch.float32), _c(k_pool, torch.bfloat16), _c(v_pool, torch.bfloat16)
    _c(positions, torch.int32), _c(slot_mapping, torch.int32), _c(cos_sin, torch.float32)
    T = positions.numel()
    nparts = parts.numel() // (T * (num_q_heads + 2 * num_kv_heads) * head_dim)
    q = torch.empty(T, num_q_heads, head_dim, dtype=torch.bfloat16, device=parts.device)
    num_slots = k_pool.numel() // (num_kv_heads * head_dim)
    check(lib().msgl_qknorm_rope_store_kv_partials(
        _p(parts), nparts, _p(q), _p(k_pool), _p(v_pool), num_slots, _p(positions),
        _p(slot_mapping), _p(cos_sin), _p(q_norm), _p(k_norm), T, num_q_heads, num_kv_heads,
        head_dim, eps, _s()))
    return q


def _mrope_args(positions, slot_mapping, cos_sin, q_norm, k_norm, k_pool, v_pool, sections, head_dim):
    """Checked [3, T] positions (any row stride): T, their row stride, the host section array."""
    _on(torch.int32, slot_mapping)
    _on(torch.float32, cos_sin)
    three, T = positions.shape
    if (three != 3 or positions.dtype != torch.int32 or positions.get_device() != slot_mapping.get_device()
            or (T > 1 and positions.stride(1) != 1)):
        raise ValueError("expected int32 positions [3, T] with contiguous rows on the current device")
    assert slot_mapping.numel() == T, "expected slot_mapping [T]"
    assert cos_sin.dim() == 2 and cos_sin.shape[1] == head_dim, "expected cos_sin [max_position, D]"
    assert q_norm.numel() == head_dim and k_norm.numel() == head_dim, "expected norm weights [D]"
    assert k_pool.numel() == v_pool.numel(), "expected pools of one size"
    return T, positions.stride(0), _SECTIONS(*sections)


def qknorm_mrope_store_kv(qkv, k_pool, v_pool, positions, slot_mapping, cos_sin, q_norm, k_norm,
                          num_q_heads, num_kv_heads, eps, sections, interleaved=False, head_dim=128,
                          out=None):
    """As qknorm_rope_store_kv with positions [3, T] (time, height, width rows) and `sections`, the
    rotary pairs of each axis (sum head_dim / 2): consecutive ranges, or interleaved."""
    if out is None:
        out = torch.empty(positions.shape[1], num_q_heads, head_dim, dtype=torch.bfloat16, device=qkv.device)
    _on(torch.bfloat16, qkv, k_pool, v_pool, q_norm, k_norm, out)
    T, stride, sec = _mrope_args(positions, slot_mapping, cos_sin, q_norm, k_norm, k_pool, v_pool, sections, head_dim)
    assert qkv.numel() == T * (num_q_heads + 2 * num_kv_heads) * head_dim, "expected qkv [T, (Hq + 2 Hkv) D]"
    assert out.numel() == T * num_q_heads * head_dim, "expected out [T, Hq, D]"
    num_slots = k_pool.numel() // (num_kv_heads * head_dim)
    check(lib().msgl_qknorm_mrope_store_kv(
        _p(qkv), _p(out), _p(k_pool), _p(v_pool), num_slots, _p(positions), stride, sec,
        int(interleaved), _p(slot_mapping), _p(cos_sin), cos_sin.shape[0], _p(q_norm), _p(k_norm), T, num_q_heads,
        num_kv_heads, head_dim, eps, _s()))
    return out


def qknorm_mrope_store_kv_partials(parts, k_pool, v_pool, positions, slot_mapping, cos_sin, q_norm,
                                   k_norm, num_q_heads, num_kv_heads, eps, sections,
                                   interleaved=False, head_dim=128, out=None):
    """As qknorm_mrope_store_kv with the QKV rows the sum of fp32 partials [P, T, (Hq+2Hkv) D]."""
    if out is None:
        out = torch.empty(positions.shape[1], num_q_heads, head_dim, dtype=torch.bfloat16, device=parts.device)
    _on(torch.float32, parts)
    _on(torch.bfloat16, k_pool, v_pool, q_norm, k_norm, out)
    T, stride, sec = _mrope_args(positions, slot_mapping, cos_sin, q_norm, k_norm, k_pool, v_pool, sections, head_dim)
    nparts = parts.shape[0]
    assert parts.numel() == nparts * T * (num_q_heads + 2 * num_kv_heads) * head_dim, "expected parts [P, T, (Hq + 2 Hkv) D]"
    assert out.numel() == T * num_q_heads * head_dim, "expected out [T, Hq, D]"
    num_slots = k_pool.numel() // (num_kv_heads * head_dim)
    check(lib().msgl_qknorm_mrope_store_kv_partials(
        _p(parts), nparts, _p(out), _p(k_pool), _p(v_pool), num_slots, _p(positions), stride, sec,
        int(interleaved), _p(slot_mapping), _p(cos_sin), cos_sin.shape[0], _p(q_norm), _p(k_norm), T,
        num_q_heads, num_kv_heads, head_dim, eps, _s()))
    return out


def decode_advance(next_tokens, input_ids, positions, slot_mapping, page_table, seq_lens,
                   free_pages, free_top, page_size=16):
    """msgl_decode_advance on device int32 tensors (in place): the next decode step's metadata."""
    for t in (next_tokens, input_ids, positions, slot_mapping, page_table, seq_lens, free_pages,
              free_top):
        _c(t, torch.int32)
    B = seq_lens.numel()
    check(lib().msgl_decode_advance(_p(next_tokens), _p(input_ids), _p(positions),
                                    _p(slot_mapping), _p(page_table), page_table.shape[1],
                                    _p(seq_lens), _p(free_pages), _p(free_top), B, page_size, _s()))


def sample(logits, temperature, top_k, top_p, seed=0, step=0, out=None):
    """msgl_sample: one token id per row of fp32 logits [B, V] (per-row parameters, device)."""
    _c(logits, torch.float32), _c(temperature, torch.float32), _c(top_k, torch.int32)
    _c(top_p, torch.float32)
    B, V = logits.shape
    if out is None:
        out = torch.empty(B, dtype=torch.int32, device=logits.device)
    check(lib().msgl_sample(_p(logits), B, V, _p(temperature), _p(top_k), _p(top_p), seed, step,
                            _p(out), _s()))
    return out


# ------------------------------------------------------------------ attention
def attention_workspace(num_reqs, max_seq_len, hq, hkv, device="cuda"):
    n = lib().msgl_paged_attention_workspace_size(num_reqs, max_seq_len, hq, hkv, 128)
    return torch.zeros(max(n, 256), dtype=torch.uint8, device=device)


def paged_attention_decode(q, k_pool, v_pool, page_table, seq_lens, max_seq_len, hq, hkv,
                           scale=None, page_size=16, workspace=None, out=None):
    _c(q, torch.bfloat16), _c(page_table, torch.int32), _c(seq_lens, torch.int32)
    B = seq_lens.numel()
    if scale is None:
        scale = 1.0 / (128 ** 0.5)
    if workspace is None:
        workspace = attention_workspace(B, max_seq_len, hq, hkv, q.device)
    if out is None:
        out = torch.empty(B, hq, 128, dtype=torch.bfloat16, device=q.device)
    num_slots = k_pool.numel() // (hkv * 128)
    check(lib().msgl_paged_attention_decode(_p(q), _p(k_pool), _p(v_pool), num_slots,
                                            _p(page_table), page_table.shape[1], _p(seq_lens), B,
                                            max_seq_len, hq, hkv, 128, page_size, scale, _p(out),
                                            _p(workspace), workspace.numel(), _s()))
    return out


def paged_attention_decode_cascade(q, k_pool, v_pool, page_table, seq_lens, max_seq_len,
                                   shared_pages, hq, hkv, scale=None, page_size=16, workspace=None,
                                   out=None):
    """msgl_paged_attention_decode_cascade: decode with the first `shared_pages` page-table
    columns common to every request."""
    _c(q, torch.bfloat16), _c(page_table, torch.int32), _c(seq_lens, torch.int32)
    B = seq_lens.numel()
    if scale is None:
        scale = 1.0 / (128 ** 0.5)
    if workspace is None:
        n = lib().msgl_paged_attention_cascade_workspace_size(B, max_seq_len, shared_pages, hq, hkv, 128)
        workspace = torch.zeros(max(n, 256), dtype=torch.uint8, device=q.device)
    if out is None:
        out = torch.empty(B, hq, 128, dtype=torch.bfloat16, device=q.device)
    num_slots = k_pool.numel() // (hkv * 128)
    check(lib().msgl_paged_attention_decode_cascade(_p(q), _p(k_pool), _p(v_pool), num_slots,
                                                    _p(page_table), page_table.shape[1],
                                                    _p(seq_lens), B, max_seq_len, shared_pages, hq,
                                                    hkv, 128, page_size, scale, _p(out),
                                                    _p(workspace), workspace.numel(), _s()))
    return out


def paged_attention_decode_noalloc(q, k_pool, v_pool, page_table, seq_lens, max_seq_len, hq, hkv,
                                   scale=None, page_size=16, out=None):
    """msgl_paged_attention_decode_noalloc: decode on the library's static scratch."""
    _c(q, torch.bfloat16), _c(page_table, torch.int32), _c(seq_lens, torch.int32)
    B = seq_lens.numel()
    if scale is None:
        scale = 1.0 / (128 ** 0.5)
    if out is None:
        out = torch.empty(B, hq, 128, dtype=torch.bfloat16, device=q.device)
    num_slots = k_pool.numel() // (hkv * 128)
    check(lib().msgl_paged_attention_decode_noalloc(_p(q), _p(k_pool), _p(v_pool), num_slots,
                                                    _p(page_table), page_table.shape[1],
                                                    _p(seq_lens), B, max_seq_len, hq, hkv, 128,
                                                    page_size, scale, _p(out), _s()))
    return out


def paged_attention_extend(q, k_pool, v_pool, page_table, seq_lens, q_indptr, max_q_len, hq, hkv,
                           scale=None, page_size=16):
    _c(q, torch.bfloat16), _c(page_table, torch.int32), _c(seq_lens, torch.int32)
    _c(q_indptr, torch.int32)
    B = seq_lens.numel()
    if scale is None:
        scale = 1.0 / (128 ** 0.5)
    out = torch.zeros_like(q)
    num_slots = k_pool.numel() // (hkv * 128)
    check(lib().msgl_paged_attention_extend(_p(q), _p(k_pool), _p(v_pool), num_slots,
                                            _p(page_table), page_table.shape[1], _p(seq_lens),
                                            _p(q_indptr), B, max_q_len, hq, hkv, 128, page_size,
                                            scale, _p(out), _s()))
    return out


# ------------------------------------------------------------------ page-sparse attention
def _rows(page_table, seq_lens, q_indptr, max_q_len, total_q):
    """Checked request metadata of the page-sparse calls: the request count."""
    _on(torch.int32, page_table, seq_lens)
    B = seq_lens.numel()
    assert page_table.dim() == 2 and page_table.shape[0] == B, "expected a page-table row per request"
    if q_indptr is None:
        assert max_q_len == 1 and total_q in (None, B), "one query row per request without q_indptr"
    else:
        _on(torch.int32, q_indptr)
        assert q_indptr.numel() == B + 1, "expected q_indptr [num_reqs + 1]"
    return B


def kv_page_bounds_(bounds, k_pool, page_table, seq_lens, num_kv_heads, q_indptr=None, max_q_len=1,
                    head_dim=128, page_size=16):
    """msgl_kv_page_bounds: smallest / largest key of the pages the last rows of each request
    touch, into bounds [num_pages, Hkv, 2, D] bf16 (in place)."""
    _on(torch.bfloat16, bounds, k_pool)
    B = _rows(page_table, seq_lens, q_indptr, max_q_len, None)
    num_slots = k_pool.numel() // (num_kv_heads * head_dim)
    assert bounds.numel() * page_size == 2 * k_pool.numel(), "expected bounds [num_pages, Hkv, 2, D]"
    check(lib().msgl_kv_page_bounds(_p(k_pool), num_slots, _p(page_table), page_table.shape[1],
                                    _p(seq_lens), _p(q_indptr), B, max_q_len, num_kv_heads,
                                    head_dim, page_size, _p(bounds), _s()))
    return bounds


def select_pages_workspace(total_q, max_seq_len, num_kv_heads, device="cuda"):
    n = lib().msgl_select_pages_workspace_size(total_q, max_seq_len, num_kv_heads)
    return torch.empty(max(n, 256), dtype=torch.uint8, device=device)


def select_pages(q, bounds, page_table, seq_lens, max_seq_len, top_pages, hq, hkv, sink_pages=1,
                 recent_pages=1, q_indptr=None, max_q_len=1, page_size=16, workspace=None, out=None):
    """msgl_select_pages: page ids [total_q, Hkv, top_pages] int32 for query rows q [total_q, Hq, D]
    (rows behind the last request: -1 unless `out` is given)."""
    _on(torch.bfloat16, q, bounds)
    T = q.numel() // (hq * 128)
    B = _rows(page_table, seq_lens, q_indptr, max_q_len, T)
    if workspace is None:
        workspace = select_pages_workspace(T, max_seq_len, hkv, q.device)
    if out is None:
        shape = (T, hkv, top_pages)
        out = (torch.empty(shape, dtype=torch.int32, device=q.device) if q_indptr is None else
               torch.full(shape, -1, dtype=torch.int32, device=q.device))
    _on(torch.int32, out)
    _on(torch.uint8, workspace)
    assert out.numel() == T * hkv * top_pages, "expected out [total_q, Hkv, top_pages]"
    check(lib().msgl_select_pages(_p(q), _p(bounds), bounds.numel() // (hkv * 256), _p(page_table),
                                  page_table.shape[1], _p(seq_lens), _p(q_indptr), B, T, max_q_len,
                                  max_seq_len, hq, hkv, 128, page_size, top_pages, sink_pages,
                                  recent_pages, _p(out), _p(workspace), workspace.numel(), _s()))
    return out


def paged_attention_pages(q, k_pool, v_pool, page_table, seq_lens, page_ids, hq, hkv, scale=None,
                          q_indptr=None, max_q_len=1, max_seq_len=None, page_size=16, out=None):
    """msgl_paged_attention_pages: attention of q [total_q, Hq, D] over the pages listed in
    page_ids [total_q, Hkv, top_pages] (select_pages, or lists of the caller's)."""
    _on(torch.bfloat16, q, k_pool, v_pool)
    _on(torch.int32, page_ids)
    T = q.numel() // (hq * 128)
    B = _rows(page_table, seq_lens, q_indptr, max_q_len, T)
    assert page_ids.dim() == 3 and page_ids.shape[:2] == (T, hkv), "expected page_ids [total_q, Hkv, top]"
    assert k_pool.numel() == v_pool.numel(), "expected pools of one size"
    if scale is None:
        scale = 1.0 / (128 ** 0.5)
    if max_seq_len is None:
        max_seq_len = page_table.shape[1] * page_size
    if out is None:
        out = torch.empty_like(q) if q_indptr is None else torch.zeros_like(q)
    _on(torch.bfloat16, out)
    assert out.numel() == q.numel(), "expected out [total_q, Hq, D]"
    num_slots = k_pool.numel() // (hkv * 128)
    check(lib().msgl_paged_attention_pages(_p(q), _p(k_pool), _p(v_pool), num_slots, _p(page_table),
                                           page_table.shape[1], _p(seq_lens), _p(q_indptr), B, T,
                                           max_q_len, max_seq_len, _p(page_ids), page_ids.shape[2],
                                           hq, hkv, 128, page_size, scale, _p(out), _s()))
    return out


# ------------------------------------------------------------------ low-rank adapters
def lora_workspace(num_tokens, K, rank, device="cuda"):
    n = lib().msgl_lora_workspace_size(num_tokens, K, rank)
    return torch.empty(max(n, 256), dtype=torch.uint8, device=device)


def _r(t, dtype):
    """A 2-D tensor with contiguous rows on the current device: its row stride."""
    if (t.dim() != 2 or t.dtype != dtype or t.get_device() != torch._C._cuda_getDevice()
            or (t.shape[1] > 1 and t.stride(1) != 1)):
        raise ValueError(f"expected {dtype} rows [T, n] on the current device, got {t.dtype} "
                         f"{tuple(t.shape)} with strides {t.stride()} on {t.device}")
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _lora(x, lora_a, lora_b, scales, adapter_ids, q_indptr, max_q_len, workspace):
    _on(torch.bfloat16, lora_a, lora_b)
    _on(torch.float32, scales)
    _on(torch.int32, adapter_ids)
    n, R, K = lora_a.shape
    assert lora_b.shape[0] == n and lora_b.shape[2] == R and scales.numel() == n and x.shape[1] == K, \
        "expected lora_a [n, rank, K], lora_b [n, N, rank], scales [n], x [T, K]"
    B = adapter_ids.numel()
    if q_indptr is None:
        assert max_q_len == 1 and B == x.shape[0], "one row per request without q_indptr"
    else:
        _on(torch.int32, q_indptr)
        assert q_indptr.numel() == B + 1, "expected q_indptr [num_reqs + 1]"
    if workspace is None:
        workspace = lora_workspace(x.shape[0], K, R, x.device)
    _on(torch.uint8, workspace)
    return (_p(x), _r(x, torch.bfloat16), _p(lora_a), _p(lora_b), _p(scales), n, _p(adapter_ids),
            _p(q_indptr), B, max_q_len), (x.shape[0], lora_b.shape[1], K, R), workspace


def lora_add(x, lora_a, lora_b, scales, adapter_ids, y, q_indptr=None, max_q_len=1, workspace=None,
             out=None):
    """msgl_lora_add: y + scales[a] * (x A[a]^T) B[a]^T, a = adapter_ids[r] of the request that owns
    the row (negative: y as it is). out may be y (in place); rows of x, y, out may be strided."""
    head, sizes, workspace = _lora(x, lora_a, lora_b, scales, adapter_ids, q_indptr, max_q_len, workspace)
    if out is None:
        out = torch.empty(y.shape, dtype=y.dtype, device=y.device) if q_indptr is None else y.clone()
    assert y.shape == out.shape == sizes[:2], "expected y / out [T, N]"
    check(lib().msgl_lora_add(*head, _p(y), _r(y, torch.bfloat16), _p(out), _r(out, torch.bfloat16),
                              *sizes, _p(workspace), workspace.numel(), _s()))
    return out


def lora_partial(x, lora_a, lora_b, scales, adapter_ids, q_indptr=None, max_q_len=1, workspace=None,
                 out=None):
    """msgl_lora_partial: fp32 [T, N] scales[a] * (x A[a]^T) B[a]^T, e.g. into the last slab of the
    partials of linear_partials."""
    head, sizes, workspace = _lora(x, lora_a, lora_b, scales, adapter_ids, q_indptr, max_q_len, workspace)
    if out is None:
        make = torch.empty if q_indptr is None else torch.zeros
        out = make(sizes[:2], dtype=torch.float32, device=x.device)
    assert out.shape == sizes[:2], "expected out [T, N]"
    check(lib().msgl_lora_partial(*head, _p(out), _r(out, torch.float32), *sizes, _p(workspace),
                                  workspace.numel(), _s()))
    return out


# ------------------------------------------------------------------ GEMMs
def gemm_workspace(M, N, K, device="cuda"):
    n = lib().msgl_gemm_workspace_size(M, N, K)
    return torch.zeros(max(n, 256), dtype=torch.uint8, device=device)


def linear(x, w, out_dtype=torch.bfloat16, workspace=None):
    """y = x W^T with W [N, K] (Linear::forward)."""
    _c(x, torch.bfloat16), _c(w, torch.bfloat16)
    N, K = w.shape
    M = x.numel() // K
    y = torch.empty(M, N, dtype=out_dtype, device=x.device)
    if workspace is None:
        workspace = gemm_workspace(M, N, K, x.device)
    check(lib().msgl_gemm_bf16(_p(x), _p(w), _p(y), M, N, K, _DT[out_dtype], _p(workspace),
                               workspace.numel(), _s()))
    return y


def gemm_partials_splits(M, N, K):
    return lib().msgl_gemm_partials_splits(M, N, K)


def linear_partials(x, w, splits=None, out=None):
    """fp32 split-K partials [S, M, N] of x W^T (sum over S = x W^T)."""
    _c(x, torch.bfloat16), _c(w, torch.bfloat16)
    N, K = w.shape
    M = x.numel() // K
    if splits is None:
        splits = gemm_partials_splits(M, N, K)
    if out is None:
        out = torch.empty(splits, M, N, dtype=torch.float32, device=x.device)
    check(lib().msgl_gemm_bf16_partials(_p(x), _p(w), _p(out), M, N, K, splits, _s()))
    return out


def pack_gate_up(w_gate_up):
    _c(w_gate_up, torch.bfloat16)
    two_i, K = w_gate_up.shape
    out = torch.empty_like(w_gate_up)
    check(lib().msgl_pack_gate_up(_p(w_gate_up), _p(out), two_i // 2, K, _s()))
    return out


def gate_up_silu(x, w_packed, workspace=None):
    _c(x, torch.bfloat16), _c(w_packed, torch.bfloat16)
    two_i, K = w_packed.shape
    M = x.numel() // K
    y = torch.empty(M, two_i // 2, dtype=torch.bfloat16, device=x.device)
    if workspace is None:
        workspace = gemm_workspace(M, two_i, K, x.device)
    check(lib().msgl_gemm_gate_up_silu(_p(x), _p(w_packed), _p(y), M, two_i // 2, K, _p(workspace),
                                       workspace.numel(), _s()))
    return y


def lm_head_argmax(x, w, workspace=None):
    _c(x, torch.bfloat16), _c(w, torch.bfloat16)
    V, K = w.shape
    M = x.numel() // K
    packed = torch.empty(M, dtype=torch.int64, device=x.device)
    ids = torch.empty(M, dtype=torch.int32, device=x.device)
    if workspace is None:
        workspace = gemm_workspace(M, V, K, x.device)
    check(lib().msgl_lm_head_argmax(_p(x), _p(w), M, V, K, _p(packed), _p(ids), _p(workspace),
                                    workspace.numel(), _s()))
    return ids


def argmax(logits):
    _c(logits)
    out = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device)
    check(lib().msgl_argmax(_p(logits), logits.shape[0], logits.shape[1], _DT[logits.dtype], _p(out), _s()))
    return out


def fill_normal_(t, seed, stream_id=0, mean=0.0, std=1.0):
    _c(t, torch.bfloat16)
    check(lib().msgl_fill_normal_bf16(_p(t), t.numel(), seed, stream_id, mean, std, _s()))
    return t


def device_error(reset=True):
    code, info = C.c_int(0), C.c_int(0)
    check(lib().msgl_device_error(C.addressof(code), C.addressof(info), int(reset), _s()))
    return code.value, info.value
