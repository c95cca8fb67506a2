"""Checked device operations with the interface of the reference's cuda_ops module.

The reference wraps its `deepseekrpc_cuda` extension in checked calls
(src/deepseekrpc/cuda_ops.py:11-50): `extension()` insists on a CUDA device and
ABI generation 2, every op returns `[value, status]`, and a nonzero device
status becomes `ValidationError` after the op completes ("tentative writes
require rollback").  This module keeps those names, arguments and error
behaviour over this package's sm_100a extension, and adds the same checked
form for the fused decode-path ops.  There is no CPU fallback: without a CUDA
device or the built extension every call raises.
"""
from __future__ import annotations

import math
from functools import lru_cache


class ValidationError(ValueError):
    """An input or device state the operation refused (the reference's ValidationError)."""


class BlockError(ValidationError):
    """A change of block tables that was done all the same, around a bad block.

    A block id outside the pool (or a count of shares that is too low) was met on the way: it
    has -1 or nothing in its place, and every other request is as asked.  `value` is what the
    call returns; its moves are to be copied as ever (paged_copy), or blocks that the other
    requests hold now miss their rows.  Where nothing has changed, plain ValidationError is raised.
    """

    def __init__(self, message, value):
        super().__init__(message)
        self.value = value


@lru_cache(maxsize=1)
def extension():
    import torch
    if not torch.cuda.is_available():
        raise RuntimeError("a real CUDA device is required; CPU inference fallback is not supported")
    from . import extension as load
    module = load()
    if module.abi_version() != 2:
        raise RuntimeError("native extension ABI does not match this source")
    return module


def _status(status):
    # the op is complete once its status is read: a nonzero code is a refusal
    code = int(status.item())
    if code:
        raise ValidationError(f"native CUDA operation rejected input/state (code {code}); "
                              "tentative writes require rollback")


def _result(result):
    value, status = result
    _status(status)
    return value


# ------------------------------------------------------------ reference ops
def sparse_attention(query, window_kv, source_kv, indices, sink, *, scale: float):
    if not math.isfinite(scale) or scale <= 0:
        raise ValidationError("invalid attention scale")
    return _result(extension().sparse_attention(query, window_kv, source_kv, indices, sink, scale))


def index_scores(query, keys, weights, indices, visible):
    return _result(extension().index_scores(query, keys, weights, indices, visible))


def decode_engram(encoded):
    return _result(extension().engram_decode(encoded))


def scatter_slots(pool, generations, slots, expected_generations, values):
    _status(extension().scatter_slots(pool, generations, slots, expected_generations, values))


# ----------------------------------------------------------- decode-path ops
def topk_select(scores, lengths, k: int, *, ids=None, id_base: int = 0, return_scores: bool = False):
    """Exact top-k per row (ids ascending, -1 padded); ties go to the lower id."""
    result = extension().topk_select(scores, lengths, k, ids, id_base, return_scores)
    _status(result[1])
    return (result[0], result[2]) if return_scores else result[0]


def indexer_decode(query, weights, index_pool, block_table, visible, score_stride: int):
    return _result(extension().indexer_decode(query, weights, index_pool, block_table, visible, score_stride))


def sparse_mla_decode(query, kv_pool, block_table, visible, topk, swa, swa_len, sink, *, scale: float):
    if not math.isfinite(scale) or scale <= 0:
        raise ValidationError("invalid attention scale")
    return _result(extension().sparse_mla_decode(query, kv_pool, block_table, visible, topk, swa, swa_len,
                                                 sink, scale))


def decode_step(idx_q, idx_w, index_pool, query, kv_pool, block_table, visible, max_visible: int, k: int,
                swa, swa_len, sink, *, scale: float, return_scores: bool = False):
    """Indexer -> exact top-k -> sparse MLA in one device chain; returns (out, topk[, scores])."""
    if not math.isfinite(scale) or scale <= 0:
        raise ValidationError("invalid attention scale")
    result = extension().decode_step(idx_q, idx_w, index_pool, query, kv_pool, block_table, visible,
                                     max_visible, k, swa, swa_len, sink, scale, return_scores)
    _status(result[2])
    return (result[0], result[1], result[3]) if return_scores else (result[0], result[1])


def append_kv_index(kv_pool, index_pool, generations, block_table, seq, positions, expected, kv_values,
                    index_values, swa=None):
    """Generation-checked append; a refused row raises ValidationError and was not written.

    Rows whose seq and position are both -1 (paged_plan's padding) are skipped."""
    _status(extension().append_kv_index(kv_pool, index_pool, generations, block_table, seq, positions,
                                        expected, kv_values, index_values, swa))


# -------------------------------------------------- around the decode path
def paged_plan(lengths, new_tokens, held, block_table, free_ring, ring_state, tokens: int, *, shares=None):
    """Blocks for every request's new tokens and the map of those tokens to pool rows.

    Updates held, block_table, free_ring and ring_state in place; returns
    (seq, positions, slots, cu_tokens, visible).  A batch whose counts are refused changes
    nothing; one that met a block id outside the pool raises too, and has -1 in its place.

    Where requests share blocks (paged_fork), one that became shorter goes through paged_release
    first: the plan would give its surplus blocks to the ring, and map its new tokens to the
    others, whoever else has them.  With `shares` such a batch is refused.
    """
    *value, status = extension().paged_plan(lengths, new_tokens, held, block_table, free_ring, ring_state, tokens,
                                            shares=shares)
    _status(status)
    return tuple(value)


def _moves(result, changed):
    """(moves, count) of a call that reports; changed(count): whether it has changed any table."""
    moves, count, status = result
    code = int(status.item())
    if code and changed(int(count.item())):
        raise BlockError(f"native CUDA operation met a bad block (code {code}); its moves are still to be copied",
                         (moves, count))
    _status(status)
    return moves, count


def paged_fork(parent, lengths, held, block_table, free_ring, ring_state, shares):
    """Requests with a parent become its first `lengths` tokens, on the parent's whole blocks.

    Updates the five tables in place; returns (moves, count), the rows of partial last
    blocks that paged_copy has to copy in every pool.  A refused batch changes nothing; one
    that is done around a bad block raises BlockError, which has the moves.
    """
    before = held.clone()
    return _moves(extension().paged_fork(parent, lengths, held, block_table, free_ring, ring_state, shares),
                  lambda count: count > 0 or not before.equal(held))


def paged_release(lengths, held, block_table, free_ring, ring_state, shares):
    """Cuts every request to `lengths` tokens; blocks that nobody maps any more are free again.

    Returns (moves, count): a partial last block that others map too is exchanged for a
    fresh one, whose rows paged_copy has to copy.  A refused batch changes nothing; one that is
    done around a bad block raises BlockError, which has the moves.  Too few free blocks for the
    exchanges is a refusal, whatever else the batch gives back: a call with the lengths rounded
    up to 64 needs none, and frees them for the one with the lengths.
    """
    before = held.clone()
    return _moves(extension().paged_release(lengths, held, block_table, free_ring, ring_state, shares),
                  lambda count: count > 0 or not before.equal(held))


def paged_compact(held, block_table, free_ring, ring_state, shares):
    """The blocks in use get the lowest ids; returns (moves, count) of the blocks to copy.

    A `held` out of range is refused, with nothing changed; a bad block id raises BlockError,
    which has the moves of the others.
    """
    return _moves(extension().paged_compact(held, block_table, free_ring, ring_state, shares),
                  lambda _: not bool(((held < 0) | (held > block_table.shape[1])).any()))


def paged_copy(pools, generations, moves, count):
    """Copies the rows of the moves in every pool [rows, width] and bumps their generations."""
    _status(extension().paged_copy(list(pools), list(generations), moves, count))


def rope(tensors, positions, frequencies, *, offsets, interleaved, mscale: float = 1.0, inverse: bool = False,
         out=None):
    """Rotates 1 to 4 tensors [tokens(, heads), width] by their positions in one launch.

    offsets and interleaved: first rotated column and layout of each tensor.  out:
    where to write (the tensors themselves rotate in place); new tensors without it,
    which carry the gradient of those that require one.  inverse: the transposed
    rotation, which is the gradient's.  There is no gradient of the frequencies, none
    through `out`, and no writing into a tensor that requires one.
    """
    import torch
    tensors = list(tensors)
    if torch.is_grad_enabled():
        if frequencies.requires_grad:
            raise ValidationError("the gradient of rotary frequencies is not provided")
        if out is None and any(t.requires_grad for t in tensors):
            from .rotary import Rotation
            return list(Rotation.apply(positions, frequencies, list(offsets), list(interleaved), mscale, inverse,
                                       True, *tensors))
    # new tensors are copies, so that padding rows keep their values
    out = [t.detach().clone() for t in tensors] if out is None else list(out)
    _status(extension().rope(tensors, out, positions, frequencies, list(offsets), list(interleaved), mscale=mscale,
                             inverse=inverse))
    return out


def tree_mla_decode(query, kv_pool, block_table, context, cu_nodes, tree_mask, max_nodes: int, *, scale: float,
                    sink=None, out=None, return_lse: bool = False):
    """Attention of drafted tokens over their request's cached rows and their own branch.

    Rows at or past cu_nodes[-1] (padding) are zeros, their lse -inf; those of `out` stay.
    """
    if not math.isfinite(scale) or scale <= 0:
        raise ValidationError("invalid attention scale")
    result = extension().tree_mla_decode(query, kv_pool, block_table, context, cu_nodes, tree_mask, max_nodes, scale,
                                         sink=sink, return_lse=return_lse, out=out)
    _status(result[1])
    return (result[0], result[2]) if return_lse else result[0]


def prefix_mla_decode(query, kv_pool, block_table, context, cu_nodes, tree_mask, max_nodes: int, prefix, holder, *,
                      scale: float, sink=None, out=None, return_lse: bool = False):
    """tree_mla_decode for requests that continue common prompts.

    The whole blocks of a request's first `prefix` positions are read through block_table's
    row `holder`, once for all requests in a row that have the same.
    """
    if not math.isfinite(scale) or scale <= 0:
        raise ValidationError("invalid attention scale")
    result = extension().prefix_mla_decode(query, kv_pool, block_table, context, cu_nodes, tree_mask, max_nodes, prefix,
                                           holder, scale, sink=sink, return_lse=return_lse, out=out)
    _status(result[1])
    return (result[0], result[2]) if return_lse else result[0]


def sample_logits(logits, temperature, top_k, top_p, min_p, uniform):
    """One token per row after temperature, top-k, top-p and min-p; returns (tokens, chances)."""
    tokens, chances, status = extension().sample_logits(logits, temperature, top_k, top_p, min_p, uniform)
    _status(status)
    return tokens, chances
