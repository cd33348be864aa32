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
from ._launch import launch, refuse_devices, vector

MAX_REQUESTS = 4096
# bits of StepTables.status
SHORT = 1        # the free stack ran out: some requests got no new blocks (their tokens without one have slot -1, the
                 # entries of block_table for them are set to -1, which the attention does not look at)
NARROW = 2       # a request needs more blocks than the table has columns (it got none, likewise)
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
    cu, lens, status = torch.empty(2 * batch + 2, dtype=torch.int32, device=device).split((batch + 1, batch, 1))
    rows = torch.empty((3 if tree else 2, num_tokens), dtype=torch.int64, device=device).unbind(0)
    return StepTables(cu, lens, rows[0], rows[1], rows[2] if tree else None, status)


def _refuse(block_table, held, free_blocks, free_count, cached_lens, new_lens, block_size, T, parents):
    """Which of step_tables' conditions on its inputs does not hold."""
    B = held.shape[0] if held.dim() == 1 else -1
    if not (vector(held, _I32, B) and vector(cached_lens, _I32, B) and vector(new_lens, _I32, B)):
        raise ValueError("step_tables: held, cached_lens and new_lens must be contiguous int32 [B]")
    if not (vector(free_blocks, _I32, free_blocks.numel()) and vector(free_count, _I32, 1)):
        raise ValueError("step_tables: free_blocks must be a contiguous int32 vector and free_count int32 [1]")
    if T < 0 or block_size < 1:
        raise ValueError("step_tables: num_tokens >= 0 and block_size >= 1")
    if B > MAX_REQUESTS:
        raise ValueError(f"step_tables: at most {MAX_REQUESTS} requests")
    if parents is not None and not vector(parents, _I32, T):
        raise ValueError("step_tables: parents must be contiguous int32 [num_tokens]")
    raise ValueError("step_tables: block_table must be int32 [B, width] with contiguous rows that do not overlap")


_I32, _I64 = torch.int32, torch.int64


def step_tables(block_table, held, free_blocks, free_count, cached_lens, new_lens, block_size, num_tokens,
                parents=None, out=None):
    """The step's StepTables for B = len(held) requests and num_tokens token rows (rows past the last token are
    padding). int32 tensors: block_table [B, width], held [B], free_blocks [F], free_count [1] are updated in place;
    cached_lens [B], new_lens [B] (negative: the request has ended), parents [num_tokens] (index within the request of
    each token's parent, -1 for one that follows the context; None: chains) are read. `out` (alloc_tables) is written
    when given."""
    T, bs = int(num_tokens), int(block_size)
    shape, strides = block_table.shape, block_table.stride()
    B = shape[0]
    if not (len(shape) == 2 and shape[1] >= 1 and block_table.dtype == _I32 and strides[1] == 1
            and (B < 2 or strides[0] >= shape[1]) and vector(held, _I32, B) and vector(cached_lens, _I32, B)
            and vector(new_lens, _I32, B) and free_blocks.dim() == 1 and vector(free_blocks, _I32, free_blocks.shape[0])
            and vector(free_count, _I32, 1) and T >= 0 and bs >= 1 and B <= MAX_REQUESTS
            and (parents is None or vector(parents, _I32, T))):
        _refuse(block_table, held, free_blocks, free_count, cached_lens, new_lens, bs, T, parents)
    dev = held.device
    if out is None:   # alloc_tables as separate tensors, which costs less host time than cutting one up
        positions = held.new_empty(T, dtype=_I64)
        out = StepTables(held.new_empty(B + 1), torch.empty_like(held), positions, torch.empty_like(positions),
                         None if parents is None else torch.empty_like(positions), torch.empty_like(free_count))
    else:
        if not (vector(out.cu, _I32, B + 1) and vector(out.seq_lens, _I32, B) and vector(out.status, _I32, 1)
                and vector(out.positions, _I64, T) and vector(out.slots, _I64, T)
                and (parents is None or (out.mask is not None and vector(out.mask, _I64, T)))):
            raise ValueError("step_tables: out does not fit (alloc_tables(B, num_tokens, parents is not None, device))")
        if parents is None and out.mask is not None:
            out = out._replace(mask=None)
    if not (dev.type == "cuda" and block_table.device == dev and cached_lens.device == dev and new_lens.device == dev
            and free_blocks.device == dev and free_count.device == dev and out.cu.device == dev
            and out.seq_lens.device == dev and out.positions.device == dev and out.slots.device == dev
            and out.status.device == dev
            and (parents is None or (parents.device == dev and out.mask.device == dev))):
        refuse_devices("step_tables", held, block_table, cached_lens, new_lens, free_blocks, free_count, parents, *out)
    if B == 0:
        out.cu.zero_()
        out.positions.zero_()
        out.slots.fill_(-1)
        out.status.zero_()
        if out.mask is not None:
            out.mask.zero_()
        return out
    launch("vt_step_tables", _build.load().vt_step_tables, dev.index, block_table.data_ptr(),
           max(strides[0], shape[1]), shape[1], held.data_ptr(), free_blocks.data_ptr(), free_blocks.shape[0],
           free_count.data_ptr(), cached_lens.data_ptr(), new_lens.data_ptr(),
           None if parents is None else parents.data_ptr(), B, T, bs, out.cu.data_ptr(), out.seq_lens.data_ptr(),
           out.positions.data_ptr(), out.slots.data_ptr(), None if out.mask is None else out.mask.data_ptr(),
           out.status.data_ptr())
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
