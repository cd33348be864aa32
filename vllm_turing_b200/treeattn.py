"""Attention of a step's new tokens over the paged cache (csrc/tree_attn.cu): single tokens, chains, and trees of
drafted tokens (up to 64 a request) whose mask words come from steptables.step_tables."""
import struct

import torch

from . import _build
from ._launch import grad_enabled, launch, need, refuse_devices, refuse_dtypes, refuse_grad, vector

MAX_NEW = 64
MAX_GROUP = 128   # query heads to a cached head


_STRIDES = struct.Struct("10q").pack   # an int64 array for the C entry
_CODE = {torch.float16: 0, torch.bfloat16: 1}
_ws_words = {}   # (device, D) -> workspace, in 32-bit words


def _workspace(index, max_new, Hq, Hkv, D):
    key = (index, D)
    n = _ws_words.get(key)
    if n is None:
        with torch.cuda.device(index):
            n = _ws_words[key] = (int(_build.load().vt_tree_attention_ws_bytes(max_new, Hq, Hkv, D)) + 3) // 4
    return n


def _aligned(c, s):
    return s[3] == 1 and (s[0] | s[1] | s[2]) & 7 == 0 and c.data_ptr() & 15 == 0


def _refuse(q, k_cache, v_cache, block_table, cu, seq_lens, max_new, mask):
    """Which of tree_attention's conditions on its inputs does not hold."""
    need(q.dim() == 3 and (q.stride(2) == 1 or q.numel() == 0), "tree_attention: q must be [T, Hq, D] with a "
                                                                "contiguous last dimension")
    T, Hq, D = q.shape
    need(D % 8 == 0 and 8 <= D <= 256, f"tree_attention: D must be a multiple of 8 up to 256, got {D}")
    need(k_cache.dim() == 4 and v_cache.shape == k_cache.shape and k_cache.shape[3] == D,
         f"tree_attention: the caches must be [num_blocks, block_size, Hkv, {D}] alike")
    nb, bs, Hkv, _ = k_cache.shape
    need(nb >= 1 and bs >= 8 and bs % 8 == 0, "tree_attention: at least one block, block_size a multiple of 8")
    need(Hkv >= 1 and Hq >= 1 and Hq % Hkv == 0 and Hq // Hkv <= MAX_GROUP,
         f"tree_attention: {Hq} query heads over {Hkv} cached heads (a multiple, at most {MAX_GROUP} to one)")
    need(_aligned(k_cache, k_cache.stride()) and _aligned(v_cache, v_cache.stride()),
         "tree_attention: caches 16-byte aligned, last dimension contiguous, other strides multiples of 8")
    need(1 <= max_new <= MAX_NEW, f"tree_attention: max_new must be 1 .. {MAX_NEW}, got {max_new}")
    B = seq_lens.shape[0] if seq_lens.dim() == 1 else -1
    need(B >= 0 and vector(seq_lens, torch.int32, B) and vector(cu, torch.int32, B + 1),
         "tree_attention: seq_lens must be contiguous int32 [B] and cu int32 [B + 1]")
    need(mask is None or vector(mask, torch.int64, T), "tree_attention: mask must be contiguous int64 [T]")
    raise ValueError("tree_attention: block_table must be int32 [B, width], width >= 1, with contiguous rows")


def tree_attention(q, k_cache, v_cache, block_table, cu, seq_lens, max_new, mask=None, scale=None, out=None):
    """out [T, Hq, D]: softmax attention of the new tokens q [T, Hq, D] of B requests over k_cache / v_cache
    [num_blocks, block_size, Hkv, D]. Request b's tokens are rows cu[b] .. cu[b + 1] - 1 (int32 [B + 1]); its cache
    holds seq_lens[b] keys (int32 [B]), the last of which are those tokens, in the blocks block_table[b] (int32 [B, W]).
    A token sees all keys before the step's own and, of those, the ones whose bit is set in its mask word (int64 [T]);
    without a mask, itself and the ones before it. A token that sees nothing gets 0. max_new (1 .. 64): the largest
    number of tokens of a request in this call. Rows of `out` past the last token are left as they were.
    The first call on a device must come before any stream capture. D % 8 == 0 up to 256, block_size % 8 == 0, Hq a
    multiple of Hkv (at most 128 times it); scale defaults to D ** -0.5. Not recorded for autograd: inputs that require a
    gradient are refused."""
    qshape, cshape, tshape = q.shape, k_cache.shape, block_table.shape
    max_new = int(max_new)
    if not (len(qshape) == 3 and len(cshape) == 4 and len(tshape) == 2):
        _refuse(q, k_cache, v_cache, block_table, cu, seq_lens, max_new, mask)
    if grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        refuse_grad("tree_attention")
    T, Hq, D = qshape
    nb, bs, Hkv, _ = cshape
    B = tshape[0]
    qs, ks, vs, ts = q.stride(), k_cache.stride(), v_cache.stride(), block_table.stride()
    if not (qs[2] == 1 and 8 <= D <= 256 and D & 7 == 0 and v_cache.shape == cshape and cshape[3] == D and nb >= 1
            and bs >= 8 and bs & 7 == 0 and 1 <= Hkv <= Hq <= MAX_GROUP * Hkv and Hq % Hkv == 0
            and _aligned(k_cache, ks) and _aligned(v_cache, vs) and 1 <= max_new <= MAX_NEW
            and vector(seq_lens, torch.int32, B) and vector(cu, torch.int32, B + 1)
            and block_table.dtype == torch.int32 and (ts[1] == 1 or tshape[1] == 1) and tshape[1] >= 1
            and (mask is None or vector(mask, torch.int64, T))) and T > 0:
        _refuse(q, k_cache, v_cache, block_table, cu, seq_lens, max_new, mask)
    dt, dev = q.dtype, q.device
    if out is None:
        out = torch.empty_like(q)
    elif not (out.shape == qshape and (out.stride()[2] == 1 or T == 0)):
        raise ValueError("tree_attention: out must have q's shape and a contiguous last dimension")
    code = _CODE.get(dt)
    if code is None or not (k_cache.dtype == dt and v_cache.dtype == dt and out.dtype == dt):
        refuse_dtypes("tree_attention", q, k_cache, v_cache, out)
    if not (dev.type == "cuda" and k_cache.device == dev and v_cache.device == dev and block_table.device == dev
            and cu.device == dev and seq_lens.device == dev and out.device == dev
            and (mask is None or mask.device == dev)):
        refuse_devices("tree_attention", q, k_cache, v_cache, block_table, cu, seq_lens, mask, out)
    if T == 0 or B == 0:
        return out
    n = _workspace(dev.index, max_new, Hq, Hkv, D)
    ws = seq_lens.new_empty(n)
    os = out.stride()
    launch("vt_tree_attention", _build.load().vt_tree_attention, dev.index, q.data_ptr(), k_cache.data_ptr(),
           v_cache.data_ptr(), out.data_ptr(),
           _STRIDES(qs[0], qs[1], os[0], os[1], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2]), block_table.data_ptr(),
           ts[0], tshape[1], cu.data_ptr(), seq_lens.data_ptr(), None if mask is None else mask.data_ptr(), B, T,
           max_new, Hq, Hkv, D, nb, bs, D ** -0.5 if scale is None else scale, code, ws.data_ptr(), 4 * n)
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
