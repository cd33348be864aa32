"""Attention of a step's new tokens over the paged cache (csrc/tree_attn.cu): single tokens, chains, and trees of
drafted tokens (up to 64 a request) whose mask words come from steptables.step_tables."""
import ctypes

import torch

from . import _build
from ._launch import dtype_code, launch, need, same_device, vector

MAX_NEW = 64


def _cache_ok(c):
    return c.stride(3) == 1 and all(s % 8 == 0 for s in c.stride()[:3]) and c.data_ptr() % 16 == 0


def tree_attention(q, k_cache, v_cache, block_table, cu, seq_lens, max_new, mask=None, scale=None, out=None):
    """out [T, Hq, D]: softmax attention of the new tokens q [T, Hq, D] of B requests over k_cache / v_cache
    [num_blocks, block_size, Hkv, D]. Request b's tokens are rows cu[b] .. cu[b + 1] - 1 (int32 [B + 1]); its cache
    holds seq_lens[b] keys (int32 [B]), the last of which are those tokens, in the blocks block_table[b] (int32 [B, W]).
    A token sees all keys before the step's own and, of those, the ones whose bit is set in its mask word (int64 [T]);
    without a mask, itself and the ones before it. A token that sees nothing gets 0. max_new (1 .. 64): the largest
    number of tokens of a request in this call. Rows of `out` past the last token are left as they were.
    D % 8 == 0 up to 256, block_size % 8 == 0, Hq a multiple of Hkv; scale defaults to D ** -0.5."""
    need(q.dim() == 3 and (q.stride(2) == 1 or q.numel() == 0), "tree_attention: q must be [T, Hq, D] with a "
                                                                "contiguous last dimension")
    T, Hq, D = q.shape
    need(D % 8 == 0 and 8 <= D <= 256, f"tree_attention: D must be a multiple of 8 up to 256, got {D}")
    need(k_cache.dim() == 4 and v_cache.shape == k_cache.shape and k_cache.shape[3] == D,
         f"tree_attention: the caches must be [num_blocks, block_size, Hkv, {D}] alike")
    nb, bs, Hkv, _ = k_cache.shape
    need(nb >= 1 and bs >= 8 and bs % 8 == 0, "tree_attention: at least one block, block_size a multiple of 8")
    need(Hkv >= 1 and Hq >= 1 and Hq % Hkv == 0, f"tree_attention: {Hq} query heads over {Hkv} cached heads")
    need(_cache_ok(k_cache) and _cache_ok(v_cache), "tree_attention: caches 16-byte aligned, last dimension "
                                                    "contiguous, other strides multiples of 8")
    max_new = int(max_new)
    need(1 <= max_new <= MAX_NEW, f"tree_attention: max_new must be 1 .. {MAX_NEW}, got {max_new}")
    B = seq_lens.shape[0] if seq_lens.dim() == 1 else -1
    need(B >= 0 and vector(seq_lens, torch.int32, B) and vector(cu, torch.int32, B + 1),
         "tree_attention: seq_lens must be contiguous int32 [B] and cu int32 [B + 1]")
    need(block_table.dim() == 2 and block_table.dtype == torch.int32 and block_table.shape[0] == B
         and (block_table.shape[1] == 1 or block_table.stride(1) == 1 or block_table.numel() == 0),
         "tree_attention: block_table must be int32 [B, width] with contiguous rows")
    need(mask is None or vector(mask, torch.int64, T), "tree_attention: mask must be contiguous int64 [T]")
    if out is None:
        out = torch.empty(T, Hq, D, dtype=q.dtype, device=q.device)
    need(out.shape == q.shape and (out.stride(2) == 1 or out.numel() == 0),
         "tree_attention: out must have q's shape and a contiguous last dimension")
    code = dtype_code("tree_attention", q, k_cache, v_cache, out)
    dev = same_device("tree_attention", q, k_cache, v_cache, block_table, cu, seq_lens, mask, out)
    if T == 0 or B == 0:
        return out
    L = _build.load()
    ws = torch.empty(L.vt_tree_attention_ws_bytes(max_new, Hq, Hkv, D), dtype=torch.uint8, device=dev)
    qs, os, ks, vs = q.stride(), out.stride(), k_cache.stride(), v_cache.stride()
    strides = (ctypes.c_longlong * 10)(qs[0], qs[1], os[0], os[1], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2])
    launch("vt_tree_attention", L.vt_tree_attention, dev, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
           out.data_ptr(), strides, block_table.data_ptr(), block_table.stride(0), block_table.shape[1], cu.data_ptr(),
           seq_lens.data_ptr(), mask.data_ptr() if mask is not None else None, B, T, max_new, Hq, Hkv, D, nb, bs,
           D ** -0.5 if scale is None else float(scale), code, ws.data_ptr(), ws.numel())
    return out


_frag = torch.library.Library("vllm_turing", "FRAGMENT")
_frag.define("tree_attention_(Tensor(a!) out, Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor cu, "
             "Tensor seq_lens, int max_new, Tensor? mask, float? scale) -> ()")


@torch.library.impl(_frag, "tree_attention_", "CUDA")
def _tree_attention_op(out, q, k_cache, v_cache, block_table, cu, seq_lens, max_new, mask, scale):
    tree_attention(q, k_cache, v_cache, block_table, cu, seq_lens, max_new, mask, scale, out)


@torch.library.register_fake("vllm_turing::tree_attention_")
def _tree_attention_fake(out, q, k_cache, v_cache, block_table, cu, seq_lens, max_new, mask, scale):
    return None
