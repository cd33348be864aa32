"""Rotary positions of query and key heads (csrc/rotary.cu): pairs by halves or interleaved, part of the head, scaled
for long contexts; alone (either direction), or in one kernel with the write of k and v to the paged cache.

Angles come from 64-bit frequencies and are reduced in 64 bits, so far positions (up to 2^31) keep 32-bit accuracy
without a table of cosines.
"""
import math
import struct
from typing import NamedTuple

import torch

from . import _build
from ._launch import grad_enabled, launch, need, refuse_devices, refuse_dtypes, refuse_grad, vector

SCALINGS = ("none", "linear", "ntk", "yarn", "llama3")
MAX_ROT = 1024


class RopeFreqs(NamedTuple):
    turns: torch.Tensor   # float64 [rot_dim / 2] on the device: turns per position of each pair
    factor: float         # multiplies the rotated values (yarn's attention factor; 1 otherwise)
    rot_dim: int


def rope_frequencies(rot_dim, base=10000.0, scaling="none", factor=1.0, original_length=None, beta_fast=32.0,
                     beta_slow=1.0, low_freq_factor=1.0, high_freq_factor=4.0, device="cuda"):
    """Frequencies base^(-2 i / rot_dim) of the rot_dim / 2 pairs, made once per model, scaled for contexts `factor`
    times original_length:
    linear: all divided by factor; ntk: base * factor^(rot_dim / (rot_dim - 2)); yarn: pairs that turn fewer than
    beta_slow times over original_length divided by factor, those above beta_fast kept, a ramp over the pairs between,
    rotated values times 0.1 ln(factor) + 1; llama3: wavelengths above original_length / low_freq_factor divided by
    factor, below original_length / high_freq_factor kept, blended by wavelength between."""
    need(isinstance(rot_dim, int) and rot_dim >= 0 and rot_dim % 2 == 0 and rot_dim <= MAX_ROT,
         f"rope_frequencies: rot_dim must be even, 0 .. {MAX_ROT}")
    need(scaling in SCALINGS, f"rope_frequencies: scaling must be one of {SCALINGS}")
    need(base > 0 and factor > 0, "rope_frequencies: base and factor must be positive")
    need(scaling not in ("yarn", "llama3") or (original_length is not None and original_length > 0),
         f"rope_frequencies: {scaling} needs original_length")
    need(scaling != "ntk" or rot_dim != 2, "rope_frequencies: ntk needs rot_dim > 2")
    need(scaling != "yarn" or base != 1.0, "rope_frequencies: yarn needs base != 1")
    need(scaling != "llama3" or high_freq_factor > low_freq_factor > 0,
         "rope_frequencies: llama3 needs high_freq_factor > low_freq_factor > 0")
    if scaling == "ntk":
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freqs = [base ** (-2.0 * i / rot_dim) for i in range(rot_dim // 2)]
    scale = 1.0
    if scaling == "linear":
        freqs = [f / factor for f in freqs]
    elif scaling == "yarn" and freqs:
        def pair_of(turns):   # the pair that makes `turns` turns over original_length
            return rot_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), rot_dim - 1)
        width = max(high - low, 0.001)
        ramp = [min(max((i - low) / width, 0.0), 1.0) for i in range(len(freqs))]
        freqs = [f / factor * r + f * (1.0 - r) for f, r in zip(freqs, ramp)]
        scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif scaling == "llama3":
        out = []
        for f in freqs:
            wave = 2 * math.pi / f
            s = (original_length / wave - low_freq_factor) / (high_freq_factor - low_freq_factor)
            s = min(max(s, 0.0), 1.0)
            out.append((1.0 - s) * f / factor + s * f)
        freqs = out
    turns = torch.tensor([f / (2 * math.pi) for f in freqs], dtype=torch.float64, device=device)
    return RopeFreqs(turns, scale, rot_dim)


_STRIDES8, _STRIDES14 = struct.Struct("8q").pack, struct.Struct("14q").pack   # int64 arrays for the C entries
_CODE = {torch.float16: 0, torch.bfloat16: 1}


def _heads(what, x, shape):
    need(x.shape == shape and (x.stride(2) == 1 or x.numel() == 0 or shape[2] == 1),
         f"{what} must be {list(shape)} with a contiguous last dimension, got {list(x.shape)} strides {x.stride()}")


def _refuse_freqs(what, freqs, positions, T, D):
    need(isinstance(freqs, RopeFreqs) and freqs.turns.dim() == 1
         and vector(freqs.turns, torch.float64, freqs.rot_dim // 2), f"{what}: freqs must come from rope_frequencies")
    need(freqs.rot_dim <= D, f"{what}: rotates {freqs.rot_dim} of {D} values")
    need(vector(positions, torch.int64, T), f"{what}: positions must be contiguous int64 [T]")


def _plain(x, shape):
    """[T, heads, D] as given, with its values side by side (what the kernel reads without looking further)."""
    return x.shape == shape and x.stride()[2] == 1


def rotary(q, k, positions, freqs, interleaved=False, transpose=False, q_out=None, k_out=None):
    """(q_out, k_out): q [T, Hq, D] and k [T, Hkv, D] (or None) with the first freqs.rot_dim values of each head
    rotated by positions (int64 [T]); the rest copied. Any token and head strides. q_out / k_out are new tensors unless
    given; they may be q and k themselves. transpose applies the transposed map: the gradient with respect to the input,
    given the gradient of the output (and, for factor 1, the rotation back). The call itself is not recorded for
    autograd, and refuses inputs that ask for it."""
    need(q is not None and q.dim() == 3, "rotary: q must be [T, heads, D]")
    if grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        refuse_grad("rotary", " (transpose=True is the gradient's map)")
    qshape = q.shape
    T, Hq, D = qshape
    if q_out is None:
        q_out = torch.empty_like(q)
    if not (_plain(q, qshape) and _plain(q_out, qshape)):
        _heads("rotary: q", q, qshape)
        _heads("rotary: q_out", q_out, qshape)
    Hkv = 0
    if k is not None:
        Hkv = k.shape[1] if k.dim() == 3 else -1
        kshape = (T, Hkv, D)
        need(Hkv >= 0, "rotary: k must be [T, heads, D]")
        if k_out is None:
            k_out = torch.empty_like(k)
        if not (_plain(k, kshape) and _plain(k_out, kshape)):
            _heads("rotary: k", k, kshape)
            _heads("rotary: k_out", k_out, kshape)
    else:
        k_out = None
    if not (isinstance(freqs, RopeFreqs) and freqs.rot_dim <= D and vector(positions, torch.int64, T)
            and vector(freqs.turns, torch.float64, freqs.rot_dim // 2)):
        _refuse_freqs("rotary", freqs, positions, T, D)
    dt, dev = q.dtype, q.device
    code = _CODE.get(dt)
    if code is None or q_out.dtype != dt or (k is not None and (k.dtype != dt or k_out.dtype != dt)):
        refuse_dtypes("rotary", q, k, q_out, k_out)
    if not (dev.type == "cuda" and positions.device == dev and freqs.turns.device == dev and q_out.device == dev
            and (k is None or (k.device == dev and k_out.device == dev))):
        refuse_devices("rotary", q, k, positions, freqs.turns, q_out, k_out)
    if T == 0 or Hq + Hkv == 0 or D == 0:
        return q_out, k_out
    qs, qo = q.stride(), q_out.stride()
    if k is not None:
        ks, ko = k.stride(), k_out.stride()
        strides = _STRIDES8(qs[0], qs[1], qo[0], qo[1], ks[0], ks[1], ko[0], ko[1])
    else:
        strides = _STRIDES8(qs[0], qs[1], qo[0], qo[1], 0, 0, 0, 0)
    launch("vt_rotary", _build.load().vt_rotary, dev.index, q.data_ptr(), q_out.data_ptr(),
           None if k is None else k.data_ptr(), None if k is None else k_out.data_ptr(), strides,
           positions.data_ptr(), freqs.turns.data_ptr(), freqs.factor, bool(interleaved), bool(transpose), T, Hq, Hkv,
           D, freqs.rot_dim, code)
    return q_out, k_out


def rotary_cache(q, k, v, positions, slots, k_cache, v_cache, freqs, interleaved=False, q_out=None):
    """q_out: q [T, Hq, D] rotated as by rotary(); k [T, Hkv, D] rotated and v [T, Hkv, D] go to rows slots (int64 [T])
    of the paged cache k_cache, v_cache [num_blocks, block_size, Hkv, D] (any strides, last dimension contiguous). A
    token whose slot is outside the cache (step_tables gives -1) writes no k and v. Slots inside it must differ."""
    need(q is not None and q.dim() == 3 and k.dim() == 3, "rotary_cache: q and k must be [T, heads, D]")
    if grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        refuse_grad("rotary_cache")
    qshape = q.shape
    T, Hq, D = qshape
    Hkv = k.shape[1]
    kshape = (T, Hkv, D)
    if q_out is None:
        q_out = torch.empty_like(q)
    if not (_plain(q, qshape) and _plain(q_out, qshape) and _plain(k, kshape) and _plain(v, kshape) and Hkv >= 1):
        _heads("rotary_cache: q", q, qshape)
        _heads("rotary_cache: q_out", q_out, qshape)
        _heads("rotary_cache: k", k, kshape)
        _heads("rotary_cache: v", v, kshape)
        need(Hkv >= 1, "rotary_cache: k and v must have a head")
    cshape, kc, vc = k_cache.shape, k_cache.stride(), v_cache.stride()
    if not (len(cshape) == 4 and v_cache.shape == cshape and cshape[1] >= 1 and cshape[2] == Hkv and cshape[3] == D
            and ((kc[3] == 1 and vc[3] == 1) or k_cache.numel() == 0)):
        raise ValueError(f"rotary_cache: the caches must be [num_blocks, block_size, {Hkv}, {D}] with a contiguous "
                         f"last dimension, got {list(cshape)} and {list(v_cache.shape)}")
    if not (isinstance(freqs, RopeFreqs) and freqs.rot_dim <= D and vector(positions, torch.int64, T)
            and vector(freqs.turns, torch.float64, freqs.rot_dim // 2)):
        _refuse_freqs("rotary_cache", freqs, positions, T, D)
    if not vector(slots, torch.int64, T):
        raise ValueError("rotary_cache: slots must be contiguous int64 [T]")
    dt, dev = q.dtype, q.device
    code = _CODE.get(dt)
    if code is None or not (k.dtype == dt and v.dtype == dt and q_out.dtype == dt and k_cache.dtype == dt
                            and v_cache.dtype == dt):
        refuse_dtypes("rotary_cache", q, k, v, k_cache, v_cache, q_out)
    if not (dev.type == "cuda" and k.device == dev and v.device == dev and positions.device == dev
            and slots.device == dev and k_cache.device == dev and v_cache.device == dev and freqs.turns.device == dev
            and q_out.device == dev):
        refuse_devices("rotary_cache", q, k, v, positions, slots, k_cache, v_cache, freqs.turns, q_out)
    if T == 0 or D == 0:
        return q_out
    qs, qo, ks, vs = q.stride(), q_out.stride(), k.stride(), v.stride()
    strides = _STRIDES14(qs[0], qs[1], qo[0], qo[1], ks[0], ks[1], vs[0], vs[1], kc[0], kc[1], kc[2], vc[0], vc[1],
                         vc[2])
    launch("vt_rotary_cache", _build.load().vt_rotary_cache, dev.index, q.data_ptr(), q_out.data_ptr(), k.data_ptr(),
           v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), strides, positions.data_ptr(), slots.data_ptr(),
           freqs.turns.data_ptr(), freqs.factor, bool(interleaved), T, Hq, Hkv, D, freqs.rot_dim, cshape[0], cshape[1],
           code)
    return q_out


_frag = torch.library.Library("vllm_turing", "FRAGMENT")
_frag.define("rotary_(Tensor(a!) q_out, Tensor(b!)? k_out, Tensor q, Tensor? k, Tensor positions, Tensor turns, "
             "float factor, bool interleaved, bool transpose) -> ()")
_frag.define("rotary_cache_(Tensor(a!) q_out, Tensor q, Tensor k, Tensor v, Tensor positions, Tensor slots, "
             "Tensor(b!) k_cache, Tensor(c!) v_cache, Tensor turns, float factor, bool interleaved) -> ()")


@torch.library.impl(_frag, "rotary_", "CUDA")
def _rotary_op(q_out, k_out, q, k, positions, turns, factor, interleaved, transpose):
    rotary(q, k, positions, RopeFreqs(turns, factor, 2 * turns.shape[0]), interleaved, transpose, q_out, k_out)


@torch.library.impl(_frag, "rotary_cache_", "CUDA")
def _rotary_cache_op(q_out, q, k, v, positions, slots, k_cache, v_cache, turns, factor, interleaved):
    rotary_cache(q, k, v, positions, slots, k_cache, v_cache, RopeFreqs(turns, factor, 2 * turns.shape[0]),
                 interleaved, q_out)


@torch.library.register_fake("vllm_turing::rotary_")
def _rotary_fake(q_out, k_out, q, k, positions, turns, factor, interleaved, transpose):
    return None


@torch.library.register_fake("vllm_turing::rotary_cache_")
def _rotary_cache_fake(q_out, q, k, v, positions, slots, k_cache, v_cache, turns, factor, interleaved):
    return None
