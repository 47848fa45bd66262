"""The shape / dtype contract of the kernels, as host-side checks on tensors (real or meta).

Both routes to the C ABI run them: the custom ops in their `select` (which is also their Meta kernel) and
the out-variant launchers that the template kernels call directly.  A violation raises ValueError before
anything is launched; what the checks let through is what the kernels' address arithmetic assumes, so a
short operand can never become an out-of-bounds device access.
"""

from __future__ import annotations

import torch
from torch import Tensor

HALF_DTYPES = (torch.float16, torch.bfloat16)  # the attention and GEMM kernels are built for both 16-bit formats
PAGE_SIZES = (16, 32, 64, 128, 256)  # tokens per KV-cache page


def require(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def same_half_dtype(tensors) -> bool:
    return tensors[0].dtype in HALF_DTYPES and all(t.dtype == tensors[0].dtype for t in tensors)


def check_gemm_operands(op: str, a: Tensor, b: Tensor, dtypes=HALF_DTYPES, what: str = "float16 or both bfloat16") -> None:
    require(a.dim() == 2 and b.dim() == 2, f"{op}: a and b must be rank 2")
    require(a.dtype in dtypes and b.dtype in dtypes and (a.dtype == b.dtype or dtypes is not HALF_DTYPES),
            f"{op}: a and b must both be {what}, got {a.dtype} and {b.dtype}")
    require(a.size(1) == b.size(1), f"{op}: K mismatch, a is {tuple(a.shape)}, b is {tuple(b.shape)} (b is [N, K])")
    require(a.size(0) > 0 and b.size(0) > 0 and a.size(1) > 0, f"{op}: empty operand")


def check_attention_operands(op: str, q: Tensor, k: Tensor, v: Tensor) -> None:
    for name, t in (("q", q), ("k", k), ("v", v)):
        require(t.dim() == 4, f"{op}: {name} must be [B, H, S, D]")
    require(same_half_dtype((q, k, v)), f"{op}: q, k, v must all be float16 or all bfloat16")
    require(q.size(3) == 128, f"{op}: head dim {q.size(3)} not supported (only 128)")
    require(k.shape == v.shape, f"{op}: k and v shapes differ")
    require(q.size(0) == k.size(0) and q.size(3) == k.size(3), f"{op}: q and k disagree on B or D")
    require(k.size(1) > 0 and q.size(1) % k.size(1) == 0, f"{op}: {q.size(1)} query heads over {k.size(1)} key/value heads")
    require(q.size(2) > 0 and k.size(2) > 0, f"{op}: empty sequence")


def check_block_table(op: str, block_table: Tensor, per_seq: Tensor, num_seqs: int, per_seq_name: str = "seq_lens") -> None:
    """block_table int32 [num_seqs, max_pages] and a per-sequence int32 vector (an int64 tensor, torch's default
    for integer data, would be read as twice as many half-sized values)."""
    require(block_table.dim() == 2 and block_table.dtype == torch.int32, f"{op}: block_table must be int32 [num_seqs, max_pages_per_seq], got {block_table.dtype} {tuple(block_table.shape)}")
    require(per_seq.dim() == 1 and per_seq.dtype == torch.int32, f"{op}: {per_seq_name} must be int32 [num_seqs], got {per_seq.dtype} {tuple(per_seq.shape)}")
    require(block_table.size(0) == num_seqs and per_seq.size(0) == num_seqs, f"{op}: block_table / {per_seq_name} rows must equal num_seqs = {num_seqs}")
    require(num_seqs > 0 and block_table.size(1) > 0, f"{op}: empty batch")


def check_paged_args(op: str, q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, seq_lens: Tensor,
                     bf16_ok: bool = False) -> None:
    require(q.dim() == 3, f"{op}: q must be [num_seqs, num_q_heads, D]")
    require(k_cache.dim() == 4 and v_cache.shape == k_cache.shape, f"{op}: k_cache / v_cache must both be [num_pages, page_size, num_kv_heads, D]")
    if bf16_ok:
        require(same_half_dtype((q, k_cache, v_cache)), f"{op}: q, k_cache, v_cache must all be float16 or all bfloat16")
    else:
        require(q.dtype == torch.float16 and k_cache.dtype == torch.float16 and v_cache.dtype == torch.float16, f"{op}: q, k_cache, v_cache must be float16")
    check_block_table(op, block_table, seq_lens, q.size(0))
    require(q.size(2) == 128 and k_cache.size(3) == 128, f"{op}: head dim must be 128")
    require(k_cache.size(1) in PAGE_SIZES, f"{op}: page size {k_cache.size(1)} not supported {PAGE_SIZES}")
    hq, hkv = q.size(1), k_cache.size(2)
    require(hkv > 0 and hq % hkv == 0 and hq // hkv in (1, 2, 4, 8, 16), f"{op}: {hq} q heads over {hkv} kv heads is not supported (ratio 1, 2, 4, 8 or 16)")
    require(k_cache.size(0) > 0, f"{op}: empty cache")


def check_decode_partials(op: str, part_acc: Tensor, part_ml: Tensor, num_seqs: int, num_q_heads: int, splits: int | None = None) -> int:
    """part_acc fp32 [S, Hq, splits, 128] and part_ml fp32 [S, Hq, splits, 2]; returns the split count."""
    require(part_acc.dim() == 4 and part_acc.dtype == torch.float32 and part_ml.dtype == torch.float32,
            f"{op}: part_acc must be fp32 [S, Hq, splits, 128], part_ml fp32 [S, Hq, splits, 2]")
    ns = part_acc.size(2) if splits is None else splits
    require(tuple(part_acc.shape) == (num_seqs, num_q_heads, ns, 128) and tuple(part_ml.shape) == (num_seqs, num_q_heads, ns, 2),
            f"{op}: part_acc must be fp32 {(num_seqs, num_q_heads, ns, 128)} and part_ml fp32 {(num_seqs, num_q_heads, ns, 2)}, got "
            f"{tuple(part_acc.shape)} and {tuple(part_ml.shape)}")
    require(1 <= ns <= 1024, f"{op}: the number of kv splits must be in [1, 1024], got {ns}")
    return ns


def check_kv_append(op: str, k_new: Tensor, v_new: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, start_pos: Tensor) -> None:
    require(k_new.dim() == 4 and k_new.shape == v_new.shape, f"{op}: k_new and v_new must both be [S, n_new, Hkv, D]")
    require(k_cache.dim() == 4 and k_cache.shape == v_cache.shape, f"{op}: k_cache and v_cache must both be [P, page, Hkv, D]")
    require(same_half_dtype((k_new, v_new, k_cache, v_cache)), f"{op}: tensors must all be float16 or all bfloat16")
    require(k_new.size(3) == 128 and k_cache.size(3) == 128, f"{op}: head dim must be 128")
    require(k_cache.size(1) in PAGE_SIZES, f"{op}: page size {k_cache.size(1)} not supported {PAGE_SIZES}")
    require(k_new.size(2) == k_cache.size(2), f"{op}: k_new and k_cache disagree on the number of kv heads")
    require(k_new.size(0) > 0 and k_new.size(1) > 0 and k_cache.size(0) > 0, f"{op}: empty k_new or cache")
    check_block_table(op, block_table, start_pos, k_new.size(0), "start_pos")


def check_paged_prefill(op: str, q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, seq_lens: Tensor) -> None:
    require(q.dim() == 4, f"{op}: q must be [num_seqs, n_new, num_q_heads, D]")
    require(k_cache.dim() == 4 and k_cache.shape == v_cache.shape, f"{op}: k_cache / v_cache must both be [num_pages, page_size, num_kv_heads, D]")
    require(same_half_dtype((q, k_cache, v_cache)), f"{op}: q, k_cache, v_cache must all be float16 or all bfloat16")
    require(q.size(3) == 128 and k_cache.size(3) == 128, f"{op}: head dim must be 128")
    require(k_cache.size(1) in PAGE_SIZES, f"{op}: page size {k_cache.size(1)} not supported {PAGE_SIZES}")
    require(k_cache.size(2) > 0 and q.size(2) % k_cache.size(2) == 0, f"{op}: {q.size(2)} q heads over {k_cache.size(2)} kv heads")
    check_block_table(op, block_table, seq_lens, q.size(0))
    require(q.size(1) > 0 and k_cache.size(0) > 0, f"{op}: empty batch")


def check_mx_operand(op: str, name: str, codes: Tensor, scales: Tensor, per_byte: int = 2) -> int:
    """codes uint8 [rows, K / per_byte] with scales uint8 [rows, K / 32]; returns K."""
    what = "[rows, K/2] (two E2M1 codes per byte)" if per_byte == 2 else "[rows, K] (one E4M3 code per byte)"
    require(codes.dim() == 2 and codes.dtype == torch.uint8, f"{op}: {name} must be uint8 {what}")
    require(scales.dim() == 2 and scales.dtype == torch.uint8, f"{op}: {name}_scale must be uint8 [rows, K/32] (E8M0)")
    K = codes.size(1) * per_byte
    require(K > 0 and K % 32 == 0, f"{op}: K={K} must be a positive multiple of 32")
    require(scales.size(0) == codes.size(0) and scales.size(1) == K // 32, f"{op}: {name}_scale shape {tuple(scales.shape)} does not match {name} {tuple(codes.shape)}")
    return K


def check_mx_pair(op: str, a: Tensor, a_scale: Tensor, b: Tensor, b_scale: Tensor, per_byte: int) -> None:
    ka = check_mx_operand(op, "a", a, a_scale, per_byte)
    kb = check_mx_operand(op, "b", b, b_scale, per_byte)
    require(ka == kb, f"{op}: a and b disagree on K ({ka} vs {kb})")
    require(a.size(0) > 0 and b.size(0) > 0, f"{op}: empty operand")


def check_mxfp6_pair(op: str, a: Tensor, a_scale: Tensor, b: Tensor, b_scale: Tensor) -> None:
    for name, codes, scales in (("a", a, a_scale), ("b", b, b_scale)):
        require(codes.dim() == 2 and codes.dtype == torch.uint8, f"{op}: {name} must be uint8 [rows, K*3/4] (packed 6-bit codes)")
        require(scales.dim() == 2 and scales.dtype == torch.uint8, f"{op}: {name}_scale must be uint8 [rows, K/32] (E8M0)")
        require(scales.size(1) > 0 and codes.size(1) == scales.size(1) * 24 and scales.size(0) == codes.size(0),
                f"{op}: {name} {tuple(codes.shape)} and {name}_scale {tuple(scales.shape)} disagree (24 code bytes per scale byte)")
    require(a.size(1) == b.size(1), f"{op}: a and b disagree on K")
    require(a.size(0) > 0 and b.size(0) > 0, f"{op}: empty operand")


FP8_DTYPES = (torch.uint8, torch.float8_e4m3fn)


def check_fp8_operands(op: str, a: Tensor, b: Tensor) -> None:
    require(a.dim() == 2 and b.dim() == 2, f"{op}: a and b must be rank 2")
    require(a.dtype in FP8_DTYPES and b.dtype in FP8_DTYPES, f"{op}: a and b must be float8_e4m3fn (or its bytes as uint8)")
    require(a.size(1) == b.size(1), f"{op}: K mismatch, a is {tuple(a.shape)}, b is {tuple(b.shape)} (b is [N, K])")
    require(a.size(1) > 0 and a.size(1) % 32 == 0, f"{op}: K={a.size(1)} must be a positive multiple of 32")
    require(a.size(0) > 0 and b.size(0) > 0, f"{op}: empty operand")


def check_quantize_input(op: str, x: Tensor) -> None:
    require(x.dim() == 2, f"{op}: x must be [rows, K]")
    require(x.dtype in (torch.float16, torch.bfloat16, torch.float32), f"{op}: dtype {x.dtype} not supported")
    require(x.size(0) > 0 and x.size(1) > 0 and x.size(1) % 32 == 0, f"{op}: K must be a positive multiple of 32")


MAX_TREE_NODES = 64  # drafted nodes per sequence: a node's set of ancestors is one 64-bit word
MAX_ROTARY_DIM = 1024


def _check_int32(op: str, name: str, t: Tensor, shape: tuple) -> None:
    require(t.dtype == torch.int32 and tuple(t.shape) == shape, f"{op}: {name} must be int32 {list(shape)}, got {t.dtype} {tuple(t.shape)}")


def check_varlen_attention(op: str, q: Tensor, k: Tensor, v: Tensor, cu_q: Tensor, cu_k: Tensor) -> None:
    require(q.dim() == 3 and k.dim() == 3 and v.dim() == 3, f"{op}: q must be [total_q, H, D], k and v [total_k, Hkv, D]")
    require(same_half_dtype((q, k, v)), f"{op}: q, k, v must all be float16 or all bfloat16")
    require(q.size(2) == 128 and k.size(2) == 128, f"{op}: head dim must be 128")
    require(k.shape == v.shape, f"{op}: k and v shapes differ")
    require(k.size(1) > 0 and q.size(1) > 0 and q.size(1) % k.size(1) == 0, f"{op}: {q.size(1)} query heads over {k.size(1)} key/value heads")
    require(0 < q.size(0) <= 1 << 24 and 0 < k.size(0) <= 1 << 24, f"{op}: q and k need 1 to 2^24 rows, got {q.size(0)} and {k.size(0)}")
    require(cu_q.dim() == 1 and 2 <= cu_q.size(0) <= 65536, f"{op}: cu_seqlens_q must be int32 [num_seqs + 1] with 1 to 65535 sequences")
    _check_int32(op, "cu_seqlens_q", cu_q, (cu_q.size(0),))
    _check_int32(op, "cu_seqlens_k", cu_k, (cu_q.size(0),))


def check_tree_attention(op: str, q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, seq_lens: Tensor, parents: Tensor) -> None:
    require(q.dim() == 4, f"{op}: q must be [num_seqs, num_nodes, num_q_heads, D]")
    require(k_cache.dim() == 4 and v_cache.shape == k_cache.shape, f"{op}: k_cache / v_cache must both be [num_pages, page_size, num_kv_heads, D]")
    require(same_half_dtype((q, k_cache, v_cache)), f"{op}: q, k_cache, v_cache must all be float16 or all bfloat16")
    require(q.size(3) == 128 and k_cache.size(3) == 128, f"{op}: head dim must be 128")
    require(k_cache.size(1) in PAGE_SIZES, f"{op}: page size {k_cache.size(1)} not supported {PAGE_SIZES}")
    hq, hkv = q.size(2), k_cache.size(2)
    require(hkv > 0 and hq > 0 and hq % hkv == 0 and hq // hkv <= 128, f"{op}: {hq} q heads over {hkv} kv heads is not supported (a multiple, up to 128)")
    require(1 <= q.size(1) <= MAX_TREE_NODES, f"{op}: {q.size(1)} nodes per sequence, supported: 1 to {MAX_TREE_NODES}")
    check_block_table(op, block_table, seq_lens, q.size(0))
    _check_int32(op, "parents", parents, (q.size(0), q.size(1)))
    require(k_cache.size(0) > 0, f"{op}: empty cache")


def check_verify_draft(op: str, target_probs: Tensor, draft_probs: Tensor | None, tokens: Tensor, parents: Tensor, uniforms: Tensor) -> None:
    require(target_probs.dim() == 3 and target_probs.dtype == torch.float32, f"{op}: target_probs must be float32 [num_seqs, num_nodes, vocab]")
    S, N, V = target_probs.shape
    require(1 <= S <= 65535 and 1 <= N <= MAX_TREE_NODES and 1 <= V <= 1 << 24,
            f"{op}: {S} sequences of {N} nodes over {V} tokens, supported: 1 to 65535, 1 to {MAX_TREE_NODES}, 1 to 2^24")
    if draft_probs is not None:
        require(draft_probs.dtype == torch.float32 and draft_probs.shape == target_probs.shape, f"{op}: draft_probs must be float32 {[S, N, V]}")
    _check_int32(op, "tokens", tokens, (S, N))
    _check_int32(op, "parents", parents, (S, N))
    require(uniforms.dtype == torch.float32 and tuple(uniforms.shape) == (S, N), f"{op}: uniforms must be float32 {[S, N]}")


def check_batch_layout(op: str, block_table: Tensor, context_lens: Tensor, new_lens: Tensor, free_pages: Tensor, page_size: int, num_tokens: int) -> None:
    check_block_table(op, block_table, context_lens, context_lens.size(0) if context_lens.dim() == 1 else -1, "context_lens")
    S = context_lens.size(0)
    require(S <= 65535 and block_table.size(1) <= 1 << 22, f"{op}: at most 65535 sequences of 2^22 pages")
    require(block_table.is_contiguous(), f"{op}: block_table is written in place and must be contiguous")
    _check_int32(op, "new_lens", new_lens, (S,))
    require(free_pages.dim() == 1 and free_pages.dtype == torch.int32 and free_pages.size(0) <= 1 << 30, f"{op}: free_pages must be int32 [num_free]")
    require(page_size in PAGE_SIZES, f"{op}: page size {page_size} not supported {PAGE_SIZES}")
    require(1 <= num_tokens <= 1 << 30, f"{op}: num_tokens must be in [1, 2^30], got {num_tokens}")


def check_rope(op: str, x: Tensor, positions: Tensor, inv_freq: Tensor, dtypes=(torch.float16, torch.bfloat16, torch.float32)) -> None:
    require(x.dim() == 3 and x.dtype in dtypes, f"{op}: x must be [tokens, heads, D] in {', '.join(str(d).removeprefix('torch.') for d in dtypes)}, got {x.dtype} {tuple(x.shape)}")
    T, H, D = x.shape
    require(T > 0 and 0 < H <= 65535 and 0 < D <= 65536, f"{op}: bad size {tuple(x.shape)}")
    check_rope_angles(op, positions, inv_freq, T, D)


def check_rope_angles(op: str, positions: Tensor, inv_freq: Tensor, tokens: int, D: int) -> None:
    _check_int32(op, "positions", positions, (tokens,))
    require(inv_freq.dim() == 1 and inv_freq.dtype in (torch.float64, torch.float32), f"{op}: inv_freq must be float64 or float32 [rotary_dim / 2]")
    R = 2 * inv_freq.size(0)
    require(0 < R <= min(D, MAX_ROTARY_DIM), f"{op}: {R} rotary elements of a head of {D} (at most {MAX_ROTARY_DIM})")


def check_rope_append(op: str, q: Tensor, k_new: Tensor, v_new: Tensor, positions: Tensor, inv_freq: Tensor, k_cache: Tensor,
                      v_cache: Tensor, slots: Tensor) -> None:
    require(q.dim() == 3 and k_new.dim() == 3 and k_new.shape == v_new.shape, f"{op}: q must be [tokens, Hq, D], k_new and v_new both [tokens, Hkv, D]")
    require(k_cache.dim() == 4 and k_cache.shape == v_cache.shape, f"{op}: k_cache and v_cache must both be [P, page, Hkv, D]")
    require(same_half_dtype((q, k_new, v_new, k_cache, v_cache)), f"{op}: tensors must all be float16 or all bfloat16")
    require(q.size(2) == 128 and k_new.size(2) == 128 and k_cache.size(3) == 128, f"{op}: head dim must be 128")
    require(k_cache.size(1) in PAGE_SIZES, f"{op}: page size {k_cache.size(1)} not supported {PAGE_SIZES}")
    T = q.size(0)
    require(0 < q.size(1) <= 65535 and 0 < k_new.size(1) <= 65535, f"{op}: bad head counts {q.size(1)} and {k_new.size(1)}")
    require(T > 0 and k_new.size(0) == T and k_cache.size(0) > 0, f"{op}: empty or unequal tokens ({T} and {k_new.size(0)}) or empty cache")
    require(k_new.size(1) == k_cache.size(2), f"{op}: k_new and k_cache disagree on the number of kv heads")
    require(k_cache.is_contiguous() and v_cache.is_contiguous(), f"{op}: k_cache and v_cache are written in place and must be contiguous")
    require(slots.dtype == torch.int64 and tuple(slots.shape) == (T,), f"{op}: slots must be int64 [tokens], got {slots.dtype} {tuple(slots.shape)}")
    check_rope_angles(op, positions, inv_freq, T, 128)
