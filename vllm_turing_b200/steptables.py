"""The tables of one serving step, built on the GPU from the requests' lengths (csrc/step_tables.cu): block-table rows
extended from a stack of free blocks, the slot map, positions, and the mask words of trees of drafted tokens. Nothing
is read back to the host, so the step can be captured in a CUDA graph and its lengths changed between replays.

    st = step_tables(block_table, held, free_blocks, free_count, cached_lens, new_lens, block_size, num_tokens, parents)
    rotary.rotary_cache(q, k, v, st.positions, st.slots, k_cache, v_cache, freqs)       # per layer
    treeattn.tree_attention(q, k_cache, v_cache, block_table, st.cu, st.seq_lens, max_new, mask=st.mask)

After verification the caller sets cached_lens to what was accepted; blocks a row already holds stay with it (held) and
are used by the next step. A request is ended with a negative entry of new_lens: its blocks return to the stack.
"""
from typing import NamedTuple, Optional

import torch

from . import _build
from ._launch import launch, need, same_device, vector

MAX_REQUESTS = 4096
# bits of StepTables.status
SHORT = 1        # the free stack ran out: some requests got no new blocks (their tokens without one have slot -1)
NARROW = 2       # a request needs more blocks than the table has columns (it got none)
TOO_MANY = 4     # more tokens than num_tokens rows
BIG_TREE = 8     # a tree of more than 64 tokens
FREE_FULL = 16   # free_blocks too small for the blocks of ended requests


class StepTables(NamedTuple):
    cu: torch.Tensor                  # int32 [B + 1]: first token row of each request
    seq_lens: torch.Tensor            # int32 [B]: cached + new
    positions: torch.Tensor           # int64 [T]; 0 past the last token
    slots: torch.Tensor               # int64 [T]; -1 past the last token and where there is no block
    mask: Optional[torch.Tensor]      # int64 [T] with parents: bit j = token j of the request is seen; else None
    status: torch.Tensor              # int32 [1]: the bits above


def alloc_tables(batch, num_tokens, tree, device):
    """Buffers for step_tables(out=...), e.g. the static ones of a captured step."""
    ints = torch.empty(2 * batch + 2, dtype=torch.int32, device=device)
    rows = torch.empty(3 if tree else 2, num_tokens, dtype=torch.int64, device=device)
    return StepTables(ints[:batch + 1], ints[batch + 1:2 * batch + 1], rows[0], rows[1], rows[2] if tree else None,
                      ints[2 * batch + 1:])


def step_tables(block_table, held, free_blocks, free_count, cached_lens, new_lens, block_size, num_tokens,
                parents=None, out=None):
    """The step's StepTables for B = len(held) requests and num_tokens token rows (rows past the last token are
    padding). int32 tensors: block_table [B, width], held [B], free_blocks [F], free_count [1] are updated in place;
    cached_lens [B], new_lens [B] (negative: the request has ended), parents [num_tokens] (index within the request of
    each token's parent, -1 for one that follows the context; None: chains) are read. `out` (alloc_tables) is written
    when given."""
    B, T = held.shape[0] if held.dim() else -1, int(num_tokens)
    i32 = torch.int32
    need(block_table.dim() == 2 and block_table.dtype == i32 and B >= 0 and block_table.shape[0] == B
         and block_table.shape[1] >= 1 and (B < 2 or block_table.stride(0) >= block_table.shape[1])
         and block_table.stride(1) == 1, "step_tables: block_table must be int32 [B, width] with contiguous rows")
    need(vector(held, i32, B) and vector(cached_lens, i32, B) and vector(new_lens, i32, B),
         "step_tables: held, cached_lens and new_lens must be contiguous int32 [B]")
    need(vector(free_blocks, i32, free_blocks.numel()) and vector(free_count, i32, 1),
         "step_tables: free_blocks must be a contiguous int32 vector and free_count int32 [1]")
    need(T >= 0 and int(block_size) >= 1, "step_tables: num_tokens >= 0 and block_size >= 1")
    need(B <= MAX_REQUESTS, f"step_tables: at most {MAX_REQUESTS} requests")
    need(parents is None or vector(parents, i32, T), "step_tables: parents must be contiguous int32 [num_tokens]")
    if out is None:
        out = alloc_tables(B, T, parents is not None, held.device)
    else:
        i64 = torch.int64
        need(vector(out.cu, i32, B + 1) and vector(out.seq_lens, i32, B) and vector(out.status, i32, 1)
             and vector(out.positions, i64, T) and vector(out.slots, i64, T)
             and (parents is None or (out.mask is not None and vector(out.mask, i64, T))),
             "step_tables: out does not fit (alloc_tables(B, num_tokens, parents is not None, device))")
        if parents is None and out.mask is not None:
            out = out._replace(mask=None)
    dev = same_device("step_tables", held, block_table, cached_lens, new_lens, free_blocks, free_count, parents,
                      out.cu, out.seq_lens, out.positions, out.slots, out.mask, out.status)
    if B == 0:
        out.cu.zero_()
        out.positions.zero_()
        out.slots.fill_(-1)
        out.status.zero_()
        if out.mask is not None:
            out.mask.zero_()
        return out
    launch("vt_step_tables", _build.load().vt_step_tables, dev, block_table.data_ptr(),
           max(block_table.stride(0), block_table.shape[1]), block_table.shape[1], held.data_ptr(),
           free_blocks.data_ptr(), free_blocks.shape[0], free_count.data_ptr(), cached_lens.data_ptr(),
           new_lens.data_ptr(), parents.data_ptr() if parents is not None else None, B, T, int(block_size),
           out.cu.data_ptr(), out.seq_lens.data_ptr(), out.positions.data_ptr(), out.slots.data_ptr(),
           out.mask.data_ptr() if out.mask is not None else None, out.status.data_ptr())
    return out


_frag = torch.library.Library("vllm_turing", "FRAGMENT")
_frag.define("step_tables_(Tensor(a!) block_table, Tensor(b!) held, Tensor(c!) free_blocks, Tensor(d!) free_count, "
             "Tensor cached_lens, Tensor new_lens, int block_size, Tensor? parents, Tensor(e!) cu, "
             "Tensor(f!) seq_lens, Tensor(g!) positions, Tensor(h!) slots, Tensor(i!)? mask, Tensor(j!) status) -> ()")


@torch.library.impl(_frag, "step_tables_", "CUDA")
def _step_tables_op(block_table, held, free_blocks, free_count, cached_lens, new_lens, block_size, parents, cu,
                    seq_lens, positions, slots, mask, status):
    step_tables(block_table, held, free_blocks, free_count, cached_lens, new_lens, block_size, positions.shape[0],
                parents, StepTables(cu, seq_lens, positions, slots, mask, status))


@torch.library.register_fake("vllm_turing::step_tables_")
def _step_tables_fake(block_table, held, free_blocks, free_count, cached_lens, new_lens, block_size, parents, cu,
                      seq_lens, positions, slots, mask, status):
    return None
