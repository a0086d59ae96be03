"""Host-side mirror of the reference's op interface over the C ABI.

Names follow the ggml ops the reference's custom-op callbacks implement:
mul_mat (cb_gemv_custom / cb_gemv_batched_custom), mul_mat_id (cb_moe_forward),
flash_attn_decode (cb_paged_attention_decode), verify_accept.  All arrays are
numpy host arrays; every call goes through libdc_b200.so.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from .blocks import (BLOCK_BYTES, GGML_TYPE_BF16, GGML_TYPE_F16, GGML_TYPE_F32, GGML_TYPE_Q4_K, GGML_TYPE_Q6_K, Q8K_BYTES, QK_K,
                     row_bytes)

ROW_TYPES = {"f32": GGML_TYPE_F32, "bf16": GGML_TYPE_BF16, "f16": GGML_TYPE_F16}
_HOST_ROWS = {"f32": np.float32, "bf16": np.uint16, "f16": np.float16}      # bf16 rows on the host: their bits


def _row_type(dtype: str) -> int:
    if dtype not in ROW_TYPES:
        raise ValueError(f"row type {dtype!r} (one of {', '.join(ROW_TYPES)})")
    return ROW_TYPES[dtype]


def _dev(p: int):
    return C.c_void_p(p) if p else None


def _vp(a: np.ndarray | None):
    return a.ctypes.data_as(C.c_void_p) if a is not None else None


class Weight:
    """Handle of a GGUF tensor resident in HBM in its native block bytes."""

    def __init__(self, ctx: "Context", handle: int, ggml_type: int, K: int, N: int, E: int):
        self.ctx, self.handle, self.type, self.K, self.N, self.E = ctx, handle, ggml_type, K, N, E

    @property
    def nbytes(self) -> int:
        return row_bytes(self.type, self.K) * self.N * self.E

    def free(self):
        if self.handle:
            self.ctx._check(_lib.lib().dc_b200_free_weight(self.ctx.handle, self.handle))
            self.handle = None


class Context:
    """One GPU, one stream (dc_b200_init)."""

    def __init__(self, device: int = 0):
        self.handle = None
        h = C.c_void_p()
        st = _lib.lib().dc_b200_init(int(device), C.byref(h))
        if st != 0:
            raise _lib.DcError(st, "dc_b200_init failed (no CPU fallback exists)")
        self.handle = h
        self.device = device

    def close(self):
        if self.handle:
            _lib.lib().dc_b200_destroy(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def last_error(self) -> str:
        return (_lib.lib().dc_b200_last_error(self.handle) or b"").decode()

    def _check(self, st: int):
        if st != 0:
            raise _lib.DcError(st, self.last_error())

    def synchronize(self):
        self._check(_lib.lib().dc_b200_synchronize(self.handle))

    def set_option(self, name: str, value: int):
        self._check(_lib.lib().dc_b200_set_option(self.handle, name.encode(), int(value)))

    # ---- weights
    def upload_weight(self, ggml_type: int, data: np.ndarray, K: int, N: int, E: int = 1) -> Weight:
        data = np.ascontiguousarray(data)
        want = row_bytes(ggml_type, K) * N * E
        if data.nbytes != want:
            raise ValueError(f"weight has {data.nbytes} bytes, expected {want}")
        ne = (C.c_int64 * 4)(K, N, E, 1)
        h = C.c_void_p()
        self._check(_lib.lib().dc_b200_upload_weight(self.handle, int(ggml_type), ne, _vp(data), C.byref(h)))
        return Weight(self, h, ggml_type, K, N, E)

    # ---- Q8_K
    def quantize_q8k(self, x: np.ndarray) -> np.ndarray:
        x = np.ascontiguousarray(np.atleast_2d(x), dtype=np.float32)
        rows, K = x.shape
        out = np.zeros((rows, K // QK_K * Q8K_BYTES), dtype=np.uint8)
        self._check(_lib.lib().dc_b200_quantize_q8k(self.handle, _vp(x), rows, K, _vp(out)))
        return out

    # ---- MUL_MAT
    def mul_mat(self, w: Weight, x: np.ndarray) -> np.ndarray:
        x = np.ascontiguousarray(np.atleast_2d(x), dtype=np.float32)
        M, K = x.shape
        if K != w.K:
            raise ValueError(f"x has K={K}, weight has K={w.K}")
        y = np.empty((M, w.N), dtype=np.float32)
        self._check(_lib.lib().dc_b200_mul_mat(self.handle, w.handle, _vp(x), M, _vp(y)))
        return y

    def mul_mat_dev(self, w: Weight, x_dev: int, M: int, y_dev: int, noalloc: bool = False):
        """Device-pointer form: x_dev [M, K] f32 and y_dev [M, N] f32 are addresses from alloc().
        noalloc=True takes the entry point whose Q8_K scratch is built into the library
        (M <= 16, K <= 16384; performs no allocation)."""
        fn = _lib.lib().dc_b200_mul_mat_dev_noalloc if noalloc else _lib.lib().dc_b200_mul_mat_dev
        self._check(fn(self.handle, w.handle, C.c_void_p(x_dev), int(M), C.c_void_p(y_dev)))

    def mul_mat_block_sums(self, w: Weight, x: np.ndarray):
        x = np.ascontiguousarray(np.atleast_2d(x), dtype=np.float32)
        M, K = x.shape
        nb = K // QK_K
        I = np.zeros((M, w.N, nb), dtype=np.int32)
        Mn = np.zeros((M, w.N, nb), dtype=np.int32) if w.type == GGML_TYPE_Q4_K else None
        self._check(_lib.lib().dc_b200_mul_mat_block_sums(self.handle, w.handle, _vp(x), M, _vp(I), _vp(Mn)))
        return I, Mn

    # ---- device buffers
    def alloc(self, nbytes: int) -> int:
        p = C.c_void_p()
        self._check(_lib.lib().dc_b200_alloc_device(self.handle, int(nbytes), C.byref(p)))
        return p.value

    def free(self, dev: int):
        self._check(_lib.lib().dc_b200_free_device(self.handle, C.c_void_p(dev)))

    def to_device(self, dev: int, a: np.ndarray):
        a = np.ascontiguousarray(a)
        self._check(_lib.lib().dc_b200_copy_to_device(self.handle, C.c_void_p(dev), _vp(a), a.nbytes))

    def from_device(self, dev: int, out: np.ndarray) -> np.ndarray:
        self._check(_lib.lib().dc_b200_copy_from_device(self.handle, _vp(out), C.c_void_p(dev), out.nbytes))
        return out

    def mul_mat_id_dev(self, router: Weight, gate: Weight, up: Weight, down: Weight, x_dev: int, T: int, top_k: int,
                       y_dev: int, ids_dev: int = 0, weights_dev: int = 0, routed_scale: float = 1.0):
        """Device-pointer form of mul_mat_id (enqueue only)."""
        self._check(_lib.lib().dc_b200_mul_mat_id_dev(self.handle, router.handle, gate.handle, up.handle, down.handle,
                                                      C.c_void_p(x_dev), int(T), int(top_k), routed_scale, C.c_void_p(y_dev),
                                                      C.c_void_p(ids_dev) if ids_dev else None,
                                                      C.c_void_p(weights_dev) if weights_dev else None))

    # ---- MUL_MAT_ID
    def mul_mat_id(self, router: Weight, gate: Weight, up: Weight, down: Weight, x: np.ndarray, top_k: int,
                   routed_scale: float = 1.0):
        """One MoE FFN layer.  Returns (y [T, hidden], ids [T, top_k], weights [T, top_k])."""
        x = np.ascontiguousarray(np.atleast_2d(x), dtype=np.float32)
        T, H = x.shape
        y = np.empty((T, H), dtype=np.float32)
        ids = np.zeros((T, top_k), dtype=np.int32)
        w = np.zeros((T, top_k), dtype=np.float32)
        self._check(_lib.lib().dc_b200_mul_mat_id(self.handle, router.handle, gate.handle, up.handle, down.handle,
                                                  _vp(x), T, top_k, routed_scale, _vp(y), _vp(ids), _vp(w)))
        return y, ids, w

    def moe_route(self, logits: np.ndarray, top_k: int, routed_scale: float = 1.0):
        logits = np.ascontiguousarray(np.atleast_2d(logits), dtype=np.float32)
        T, E = logits.shape
        ids = np.zeros((T, top_k), dtype=np.int32)
        w = np.zeros((T, top_k), dtype=np.float32)
        self._check(_lib.lib().dc_b200_moe_route(self.handle, _vp(logits), T, E, top_k, routed_scale, _vp(ids), _vp(w)))
        return ids, w

    # ---- sampling / verify
    def argmax(self, logits: np.ndarray) -> np.ndarray:
        logits = np.ascontiguousarray(np.atleast_2d(logits), dtype=np.float32)
        out = np.zeros(logits.shape[0], dtype=np.int32)
        self._check(_lib.lib().dc_b200_argmax(self.handle, _vp(logits), logits.shape[0], logits.shape[1], _vp(out)))
        return out

    def softmax(self, logits: np.ndarray, temperature: float) -> np.ndarray:
        logits = np.ascontiguousarray(np.atleast_2d(logits), dtype=np.float32)
        out = np.empty_like(logits)
        self._check(_lib.lib().dc_b200_softmax(self.handle, _vp(logits), logits.shape[0], logits.shape[1],
                                               temperature, _vp(out)))
        return out

    def verify_uniforms(self, seed: int, step: int, n: int) -> np.ndarray:
        out = np.zeros(n, dtype=np.float32)
        self._check(_lib.lib().dc_b200_verify_uniforms(self.handle, seed, step, n, _vp(out)))
        return out

    def verify_accept(self, target_logits: np.ndarray, draft_tokens, draft_probs=None, uniforms=None, seed: int = 0,
                      step: int = 0, mode: int = 0, temperature: float = 1.0):
        """Returns (n_accepted, next_token)."""
        tl = np.ascontiguousarray(target_logits, dtype=np.float32)
        gamma, vocab = tl.shape[0] - 1, tl.shape[1]
        dt = np.ascontiguousarray(draft_tokens, dtype=np.int32)
        dp = np.ascontiguousarray(draft_probs, dtype=np.float32) if draft_probs is not None else None
        u = np.ascontiguousarray(uniforms, dtype=np.float32) if uniforms is not None else None
        n, t = C.c_int(0), C.c_int(0)
        self._check(_lib.lib().dc_b200_verify_accept(self.handle, _vp(tl), _vp(dt), _vp(dp), _vp(u), seed, step,
                                                     gamma, vocab, mode, temperature, C.byref(n), C.byref(t)))
        return n.value, t.value

    def sample_rows_dev(self, logits: int, rows: int, vocab: int, temperature: int, top_k: int, top_p: int, min_p: int, uniforms: int, tokens: int, p: int = 0,
                        dist: int = 0, ld: int = 0, dtype: str = "f32"):
        """One token a row from device-resident logits; settings and results are device addresses (settings 0: not used), enqueue only."""
        self._check(_lib.lib().dc_b200_sample_rows_dev(self.handle, _dev(logits), _row_type(dtype), rows, vocab, ld, _dev(temperature), _dev(top_k), _dev(top_p),
                                                       _dev(min_p), _dev(uniforms), _dev(tokens), _dev(p), _dev(dist)))

    def sample_rows(self, logits: np.ndarray, uniforms, temperature=None, top_k=None, top_p=None, min_p=None, want_dist: bool = False):
        """One token a row by temperature, top-k, top-p and min-p (scalars or one value a row).  Returns (tokens, probabilities[, distributions])."""
        logits = np.ascontiguousarray(np.atleast_2d(logits), dtype=np.float32)
        rows, vocab = logits.shape

        def per_row(v, t):
            return None if v is None else np.ascontiguousarray(np.broadcast_to(np.asarray(v, dtype=t), (rows,)))

        s = [per_row(temperature, np.float32), per_row(top_k, np.int32), per_row(top_p, np.float32), per_row(min_p, np.float32), per_row(uniforms, np.float32)]
        tokens, p = np.zeros(rows, dtype=np.int32), np.zeros(rows, dtype=np.float32)
        dist = np.empty_like(logits) if want_dist else None
        self._check(_lib.lib().dc_b200_sample_rows(self.handle, _vp(logits), rows, vocab, *(_vp(x) for x in s), _vp(tokens), _vp(p), _vp(dist)))
        return (tokens, p, dist) if want_dist else (tokens, p)

    # ---- adapters
    def lora(self, K: int, N: int, max_adapters: int, max_rank: int, dtype: str = "bf16") -> "LoraSet":
        """Low-rank adapters of a matrix of N x K; dtype: type of their matrices ("bf16", "f16")."""
        return LoraSet(self, K, N, max_adapters, max_rank, dtype)

    def lora_add_dev(self, lora: "LoraSet", x: int, M: int, ids: int, y: int, base_dev: int = 0, ld_x: int = 0, ld_base: int = 0, ld_y: int = 0):
        """y = base + each row's adapter of x (base 0: y holds it); device addresses, enqueue only."""
        self._check(_lib.lib().dc_b200_lora_add_dev(self.handle, lora.handle, _dev(x), ld_x, M, _dev(ids), _dev(base_dev), ld_base, _dev(y), ld_y))

    def mul_mat_lora_dev(self, w: Weight, lora: "LoraSet", x: int, M: int, ids: int, y: int):
        """mul_mat_dev with each row's adapter on top."""
        self._check(_lib.lib().dc_b200_mul_mat_lora_dev(self.handle, w.handle, lora.handle, _dev(x), M, _dev(ids), _dev(y)))

    # ---- paged KV
    def kv_cache(self, n_layer: int, n_kv_head: int, head_dim: int, max_blocks: int, max_seqs: int,
                 max_blocks_per_seq: int) -> "KVCache":
        return KVCache(self, n_layer, n_kv_head, head_dim, max_blocks, max_seqs, max_blocks_per_seq)

    def kv_cache_q4(self, n_layer: int, n_head: int, n_kv_head: int, head_dim: int, max_blocks: int, max_seqs: int, max_blocks_per_seq: int,
                    dtype: str = "f32") -> "KVCacheQ4":
        """Cache in 4 bits for layers of n_head query heads; dtype: rows of queries, keys, values and results ("f32", "bf16")."""
        return KVCacheQ4(self, n_layer, n_head, n_kv_head, head_dim, max_blocks, max_seqs, max_blocks_per_seq, dtype)


class LoraSet:
    """Adapters of one matrix for many requests (dc_b200_lora_*)."""

    def __init__(self, ctx: Context, K: int, N: int, max_adapters: int, max_rank: int, dtype: str = "bf16"):
        self.handle = None
        self.ctx, self.K, self.N, self.dtype = ctx, K, N, dtype
        h = C.c_void_p()
        ctx._check(_lib.lib().dc_b200_lora_create(ctx.handle, K, N, max_adapters, max_rank, _row_type(dtype), C.byref(h)))
        self.handle = h

    def close(self):
        if self.handle:
            _lib.lib().dc_b200_lora_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            if self.ctx.handle:
                self.close()
        except Exception:
            pass

    def set(self, slot: int, A: np.ndarray, B: np.ndarray, scale: float = 1.0):
        """A [rank, K] and B [N, rank]: float16 for "f16", bits (uint16) for "bf16"."""
        t = _HOST_ROWS[self.dtype]
        if A.dtype != t or B.dtype != t:
            raise ValueError(f"matrices of type {A.dtype}, {B.dtype}; {np.dtype(t)} is wanted")
        if A.ndim != 2 or A.shape[1] != self.K or B.shape != (self.N, A.shape[0]):
            raise ValueError(f"matrices of shape {A.shape}, {B.shape} beside one of {self.N} x {self.K}")
        A, B = np.ascontiguousarray(A), np.ascontiguousarray(B)
        self.ctx._check(_lib.lib().dc_b200_lora_set(self.handle, slot, A.shape[0], _vp(A), _vp(B), scale))

    def set_dev(self, slot: int, rank: int, A: int, B: int, scale: float = 1.0):
        """The same from device addresses, enqueue only."""
        self.ctx._check(_lib.lib().dc_b200_lora_set_dev(self.handle, slot, rank, _dev(A), _dev(B), scale))

    def clear(self, slot: int):
        self.ctx._check(_lib.lib().dc_b200_lora_set_dev(self.handle, slot, 0, None, None, 0.0))


class KVCache:
    """Paged fp16 KV cache with 16-token blocks (dc_b200_kv_*)."""

    def __init__(self, ctx: Context, n_layer, n_kv_head, head_dim, max_blocks, max_seqs, max_blocks_per_seq):
        self.ctx, self.n_layer, self.n_kv, self.head_dim = ctx, n_layer, n_kv_head, head_dim
        h = C.c_void_p()
        ctx._check(_lib.lib().dc_b200_kv_create(ctx.handle, n_layer, n_kv_head, head_dim, max_blocks, max_seqs,
                                                max_blocks_per_seq, C.byref(h)))
        self.handle = h

    def close(self):
        if self.handle:
            _lib.lib().dc_b200_kv_destroy(self.handle)
            self.handle = None

    def seq_alloc(self) -> int:
        s = C.c_int(-1)
        self.ctx._check(_lib.lib().dc_b200_kv_seq_alloc(self.handle, C.byref(s)))
        return s.value

    def seq_free(self, seq: int):
        self.ctx._check(_lib.lib().dc_b200_kv_seq_free(self.handle, seq))

    def seq_reserve(self, seq: int, n_tokens: int):
        self.ctx._check(_lib.lib().dc_b200_kv_seq_reserve(self.handle, seq, n_tokens))

    def block_table(self, seq: int) -> np.ndarray:
        n = C.c_int(0)
        self.ctx._check(_lib.lib().dc_b200_kv_block_table(self.handle, seq, None, 0, C.byref(n)))
        out = np.zeros(max(n.value, 1), dtype=np.int32)
        self.ctx._check(_lib.lib().dc_b200_kv_block_table(self.handle, seq, _vp(out), out.size, C.byref(n)))
        return out[:n.value]

    def free_blocks(self) -> int:
        return _lib.lib().dc_b200_kv_free_blocks(self.handle)

    def read_block(self, layer: int, block: int):
        shape = (16, self.n_kv, self.head_dim)
        k = np.zeros(shape, dtype=np.float16)
        v = np.zeros(shape, dtype=np.float16)
        self.ctx._check(_lib.lib().dc_b200_kv_read_block(self.handle, layer, block, _vp(k), _vp(v)))
        return k, v

    def flash_attn_decode(self, layer: int, q, k, v, seq_ids, positions, scale: float) -> np.ndarray:
        """Writes the tokens' K/V at their positions, then attends.  q [T, n_head, hd]; k, v [T, n_kv, hd]."""
        q = np.ascontiguousarray(q, dtype=np.float32)
        k = np.ascontiguousarray(k, dtype=np.float32)
        v = np.ascontiguousarray(v, dtype=np.float32)
        T, n_head = q.shape[0], q.shape[1]
        seq_ids = np.ascontiguousarray(seq_ids, dtype=np.int32)
        positions = np.ascontiguousarray(positions, dtype=np.int32)
        out = np.empty((T, n_head, self.head_dim), dtype=np.float32)
        self.ctx._check(_lib.lib().dc_b200_flash_attn_decode(self.ctx.handle, self.handle, layer, _vp(q), _vp(k), _vp(v),
                                                             _vp(seq_ids), _vp(positions), T, n_head, scale, _vp(out)))
        return out

    def flash_attn_prefill(self, layer: int, q, k, v, seq: int, pos0: int, scale: float) -> np.ndarray:
        """Prompt chunk of one sequence: writes K/V at positions pos0.., then causal attention on the tensor cores."""
        q = np.ascontiguousarray(q, dtype=np.float32)
        k = np.ascontiguousarray(k, dtype=np.float32)
        v = np.ascontiguousarray(v, dtype=np.float32)
        n, n_head = q.shape[0], q.shape[1]
        out = np.empty((n, n_head, self.head_dim), dtype=np.float32)
        self.ctx._check(_lib.lib().dc_b200_flash_attn_prefill(self.ctx.handle, self.handle, layer, _vp(q), _vp(k), _vp(v), seq,
                                                              pos0, n, n_head, scale, _vp(out)))
        return out


class KVCacheQ4(KVCache):
    """Paged KV cache in 4 bits (dc_b200_kv_create_q4); sequences, forks and block tables as in KVCache."""

    def __init__(self, ctx: Context, n_layer, n_head, n_kv_head, head_dim, max_blocks, max_seqs, max_blocks_per_seq, dtype="f32"):
        self.handle = None
        self.ctx, self.n_layer, self.n_head, self.n_kv, self.head_dim, self.dtype = ctx, n_layer, n_head, n_kv_head, head_dim, dtype
        self.n_tokens = 0
        h = C.c_void_p()
        ctx._check(_lib.lib().dc_b200_kv_create_q4(ctx.handle, n_layer, n_head, n_kv_head, head_dim, _row_type(dtype), max_blocks, max_seqs,
                                                   max_blocks_per_seq, C.byref(h)))
        self.handle = h

    def __del__(self):
        try:
            if self.ctx.handle:
                self.close()
        except Exception:
            pass

    def seq_fork(self, seq: int) -> int:
        """New sequence sharing seq's blocks (copy-on-write)."""
        s = C.c_int(-1)
        self.ctx._check(_lib.lib().dc_b200_kv_seq_fork(self.handle, seq, C.byref(s)))
        return s.value

    def batch(self, seqs, pos0, counts):
        """Begins a step: counts[e] new tokens of seqs[e] from position pos0[e] on."""
        a = [np.ascontiguousarray(x, dtype=np.int32).reshape(-1) for x in (seqs, pos0, counts)]
        if not a[0].size == a[1].size == a[2].size:
            raise ValueError("seqs, pos0 and counts differ in length")
        self.ctx._check(_lib.lib().dc_b200_kv_batch(self.handle, a[0].size, *(_vp(x) for x in a)))
        self.n_tokens = int(a[2].sum())

    def write_dev(self, layer: int, k: int, v: int, ld: int = 0, k_held: int = 0, v_held: int = 0):
        """Writes the step's rows (device addresses) into one layer."""
        self.ctx._check(_lib.lib().dc_b200_kv_q4_write_dev(self.ctx.handle, self.handle, layer, _dev(k), _dev(v), ld, _dev(k_held), _dev(v_held)))

    def attend_dev(self, layer: int, q: int, k: int, v: int, scale: float, out: int, ld_q: int = 0, ld_kv: int = 0, ld_out: int = 0, k_held: int = 0,
                   v_held: int = 0):
        """Writes the step's rows (k = v = 0: they stand there already), then attends; device addresses, enqueue only."""
        self.ctx._check(_lib.lib().dc_b200_flash_attn_q4_dev(self.ctx.handle, self.handle, layer, _dev(q), ld_q, _dev(k), _dev(v), ld_kv, scale, _dev(out),
                                                             ld_out, _dev(k_held), _dev(v_held)))

    def attend(self, layer: int, q, k, v, scale: float) -> np.ndarray:
        """The same on host arrays: q [T, n_head, hd], k and v [T, n_kv, hd] (both None: written already); bf16 rows as their bits (uint16)."""
        t = _HOST_ROWS[self.dtype]
        q = np.ascontiguousarray(q, dtype=t)
        if q.shape != (self.n_tokens, self.n_head, self.head_dim):
            raise ValueError(f"q has shape {q.shape}, the step has {self.n_tokens} tokens")
        k, v = (None if x is None else np.ascontiguousarray(x, dtype=t) for x in (k, v))
        for x in (k, v):
            if x is not None and x.shape != (self.n_tokens, self.n_kv, self.head_dim):
                raise ValueError(f"keys or values have shape {x.shape}, the step has {self.n_tokens} tokens")
        out = np.empty_like(q)
        self.ctx._check(_lib.lib().dc_b200_flash_attn_q4(self.ctx.handle, self.handle, layer, _vp(q), _vp(k), _vp(v), scale, _vp(out)))
        return out

    def read_block(self, layer: int, block: int):
        """The values that a block stands for: K and V, [16, n_kv, hd] f32."""
        k = np.zeros((16, self.n_kv, self.head_dim), dtype=np.float32)
        v = np.zeros_like(k)
        self.ctx._check(_lib.lib().dc_b200_kv_q4_read_block(self.handle, layer, block, _vp(k), _vp(v)))
        return k, v
