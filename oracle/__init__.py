"""CPU oracle for the DeepSeekRPC attention hot path -- TEST INFRASTRUCTURE ONLY.

This package restates the reference's CPU equations (numpy, float32, same
operation order) without the reference's fixture-size bounds, so that the B200
kernels can be checked at the BASELINE geometries.  It is the checker, never the
thing measured or shipped: only tests/, __graft_entry__.smoke() and bench.py's
CPU-baseline leg (`cpu_baseline`, `--impl reference`) may import it.  The
product package (deepseekrpc_b200) never imports it and has no CPU fallback.

Parity pinning: tests/golden/*.npz hold outputs of the reference's own
functions (src/deepseekrpc/reference_attention.py, index_selection.merge_ranked,
engram_storage.decode_fp8_rows, cache_pool.SlotMap) generated by
tests/golden/make_golden.py; tests/test_oracle_golden.py checks this oracle
against them bit for bit.
"""
from .ops import (  # noqa: F401
    bf16_bits_to_f32,
    candidate_blocks,
    candidate_positions,
    decode_step,
    engram_decode,
    f32_to_bf16_bits,
    gather_rows,
    index_scores,
    merge_ranked,
    scatter_slots,
    sparse_attention,
    tiled_topk,
)
from .append import append_kv_index, append_kv_index_ring, paged_rows, ring_rows  # noqa: F401
from .pool import PoolOracle, ReferenceRowPool  # noqa: F401
from . import serving  # noqa: F401
