"""`Hip`: the op-level backend, a Python mirror of `bobcat_metal::Metal`.

Method names, argument order and meaning follow the Metal backend
(crates/bobcat-metal/src/backend.rs:1027-2699), so the kernel tests read like
the reference's own tests (crates/bobcat/tests/metal_*.rs).  Every call goes
through the C ABI of libbobcat_hip.so; errors raise `BobcatError` carrying
the bch_status code of the matching `bobcat_metal::Error` variant.
"""
from __future__ import annotations

import ctypes as C
import weakref
from array import array
from dataclasses import dataclass
from enum import IntEnum

import numpy as np

from ._lib import BobcatError, KvShape, LogitRules, Norm as _Norm, ProfileEntry, STATUS, View as _View, check, lib


class Format(IntEnum):
    """Weight formats; values are ggml type ids (bobcat-gguf/src/lib.rs:137-148)."""
    F32 = 0
    F16 = 1
    Q4_0 = 2
    Q8_0 = 8
    Q4K = 12
    Q5K = 13
    Q6K = 14
    BF16 = 30


class Store(IntEnum):
    """bobcat_metal::Store (backend.rs:360-370)."""
    OVERWRITE = 0
    ACCUMULATE = 1
    SWIGLU = 2


class Buffer:
    """A device buffer (bobcat_metal::Buffer, backend.rs:302-325)."""

    def __init__(self, hip: "Hip", handle: int, length: int):
        self.hip = hip
        self.handle = handle
        self.len = length

    def at(self, offset: int) -> "ViewRef":
        return ViewRef(self, offset)

    def floats(self, index: int) -> "ViewRef":
        return ViewRef(self, 4 * index)

    @property
    def device_ptr(self) -> int:
        return lib().bch_buffer_device_ptr(self.handle)

    def free(self) -> None:
        if self.handle:
            lib().bch_buffer_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


@dataclass(frozen=True)
class ViewRef:
    """A position inside a buffer (bobcat_metal::View, backend.rs:337-341)."""
    buffer: Buffer
    offset: int

    def c(self) -> _View:
        return _View(self.buffer.handle, self.offset)


@dataclass(frozen=True)
class NormSpec:
    """bobcat_metal::Norm (backend.rs:344-350)."""
    weight: ViewRef
    eps: float

    def c(self) -> _Norm:
        return _Norm(self.weight.c(), self.eps)


def _view(v: ViewRef) -> _View:
    return v.c()


class KvFormat(IntEnum):
    """What a paged cache keeps a row as (bch_kv_format)."""
    F16 = 0
    I8 = 1
    F8 = 2


# One row's rules (bch_logit_row), as an array's type; NO_MASK in `mask` is no mask.
LOGIT_ROW = np.dtype([("history_at", "<u4"), ("history_len", "<u4"), ("bias_at", "<u4"), ("bias_len", "<u4"),
                      ("mask", "<u4"), ("repeat", "<f4"), ("presence", "<f4"), ("frequency", "<f4")])
NO_MASK = 0xFFFFFFFF


def kv_shape(fmt, n_kv_heads: int, head_dim: int, page_size: int, n_pages: int) -> KvShape:
    """A paged cache's shape; `fmt` a KvFormat or its name in lower case."""
    return KvShape(KvFormat[fmt.upper()] if isinstance(fmt, str) else int(fmt), n_kv_heads, head_dim, page_size, n_pages)


def kv_page_bytes(shape: KvShape) -> int:
    """Bytes of one page; 0 for a shape that is not supported."""
    return lib().bch_kv_page_bytes(C.byref(shape))


def _u32(lists, what: str) -> np.ndarray:
    """The whole numbers below 2^32 of lists or arrays, one behind the other, as the library takes them."""
    out = array("I")  # (refuses others)
    try:
        for numbers in lists:
            out.extend(numbers.tolist() if isinstance(numbers, np.ndarray) else numbers)
    except (TypeError, OverflowError) as e:
        raise ValueError(f"{what} are whole numbers below 2^32") from e
    return np.frombuffer(out, np.uint32) if out else np.empty(0, np.uint32)


def _batch(shape: KvShape, n_past, n_new, pages):
    """A batch's arguments: lengths, and each sequence's pages one list after the other."""
    past, new = (_u32([[n] if isinstance(n, (int, np.integer)) else n], "lengths") for n in (n_past, n_new))
    if past.shape != new.shape:
        raise ValueError("n_past and n_new hold one number for each sequence")
    # (The library sees one list and would deal it out anew.)
    page, pages = max(shape.page_size, 1), [seq if hasattr(seq, "__len__") else list(seq) for seq in pages]
    need, have = [-(-(p + n) // page) for p, n in zip(past.tolist(), new.tolist())], [len(seq) for seq in pages]
    if need != have:
        if len(need) != len(have):
            raise BobcatError(STATUS["Argument"], f"{len(have)} lists of pages for {len(need)} sequences")
        at = next(i for i in range(len(need)) if need[i] != have[i])
        raise BobcatError(STATUS["Argument"], f"sequence {at} needs {need[at]} pages, got {have[at]}")
    flat = _u32(pages, "pages")
    return past, new, flat, (past.size, past.ctypes.data, new.ctypes.data, flat.ctypes.data, flat.size)


def kv_plan_check(shape: KvShape, n_heads: int, n_past, n_new, pages) -> None:
    """Raise what KvPlan and its set() would, without a device."""
    *_keep, args = _batch(shape, n_past, n_new, pages)
    check(lib().bch_kv_plan_check(C.byref(shape), n_heads, *args))


class KvPlan:
    """A batch of sequences over a paged cache (bch_kv_plan)."""

    def __init__(self, hip: "Hip", shape: KvShape, n_heads: int):
        h = C.c_void_p()
        check(lib().bch_kv_plan_new(hip.handle, C.byref(shape), n_heads, C.byref(h)))
        self.handle, self.shape, self.n_heads = h.value, shape, n_heads
        hip._dependents.add(self)

    def set(self, n_past, n_new, pages) -> None:
        """The batch: past positions and new tokens of each sequence, and each sequence's list of pages
        (ceil((past + new) / page_size) of them)."""
        *_keep, args = _batch(self.shape, n_past, n_new, pages)
        check(lib().bch_kv_plan_set(self.handle, *args))

    def close(self) -> None:
        if self.handle:
            lib().bch_kv_plan_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Hip:
    """One device context with one stream (Metal::open, backend.rs:1083)."""

    def __init__(self):
        handle = C.c_void_p()
        check(lib().bch_open(C.byref(handle)))
        self.handle = handle.value
        self._buffers: list[Buffer] = []
        # Objects that hold device state of this context (model drivers);
        # they close before the context does.
        self._dependents = weakref.WeakSet()

    def close(self) -> None:
        if self.handle:
            for d in list(self._dependents):
                d.close()
            for b in self._buffers:
                b.free()
            lib().bch_close(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def device_info(self) -> tuple[str, int]:
        name = C.create_string_buffer(256)
        cus = C.c_uint32()
        check(lib().bch_device_info(self.handle, name, 256, C.byref(cus)))
        return name.value.decode(), cus.value

    # -- buffers ---------------------------------------------------------
    def new_buffer(self, length: int) -> Buffer:
        h = C.c_void_p()
        check(lib().bch_buffer_new(self.handle, length, C.byref(h)))
        b = Buffer(self, h.value, length)
        self._buffers.append(b)
        return b

    def buffer_from(self, array: np.ndarray) -> Buffer:
        a = np.ascontiguousarray(array)
        h = C.c_void_p()
        check(lib().bch_buffer_from_host(self.handle, a.ctypes.data, a.nbytes, C.byref(h)))
        b = Buffer(self, h.value, a.nbytes)
        self._buffers.append(b)
        return b

    def write(self, view: ViewRef, data: np.ndarray) -> None:
        a = np.ascontiguousarray(data)
        check(lib().bch_write(self.handle, _view(view), a.ctypes.data, a.nbytes))

    def read(self, view: ViewRef, out: np.ndarray) -> np.ndarray:
        assert out.flags.c_contiguous
        check(lib().bch_read(self.handle, _view(view), out.ctypes.data, out.nbytes))
        return out

    # -- recording -------------------------------------------------------
    def begin(self) -> None:
        check(lib().bch_begin(self.handle))

    def discard(self) -> None:
        lib().bch_discard(self.handle)

    def barrier(self) -> None:
        lib().bch_barrier(self.handle)

    def commit(self) -> int:
        t = C.c_uint64()
        check(lib().bch_commit(self.handle, C.byref(t)))
        return t.value

    def wait(self, ticket: int) -> float:
        s = C.c_double()
        check(lib().bch_wait(self.handle, ticket, C.byref(s)))
        return s.value

    def end(self) -> float:
        s = C.c_double()
        check(lib().bch_end(self.handle, C.byref(s)))
        return s.value

    def set_profiling(self, enabled: bool) -> None:
        lib().bch_set_profiling(self.handle, int(enabled))

    def profile(self) -> list[dict]:
        out = []
        for i in range(lib().bch_profile_count(self.handle)):
            e = ProfileEntry()
            check(lib().bch_profile_get(self.handle, i, C.byref(e)))
            out.append(dict(name=e.name.decode(), n_rows=e.n_rows, n_cols=e.n_cols, calls=e.calls,
                            seconds=e.seconds, bytes=e.bytes))
        return out

    # -- ops ---------------------------------------------------------------
    def dequantize(self, fmt, weights, n_rows, n_cols, out):
        check(lib().bch_dequantize(self.handle, int(fmt), _view(weights), n_rows, n_cols, _view(out)))

    def matvec(self, fmt, weights, n_rows, n_cols, x, y, norm: NormSpec | None = None,
               accumulate: bool = False):
        n = C.byref(norm.c()) if norm is not None else None
        check(lib().bch_matvec(self.handle, int(fmt), _view(weights), n_rows, n_cols, _view(x),
                               _view(y), n, int(accumulate)))

    def matvec_swiglu(self, fmt, gate, up, n_rows, n_cols, x, norm: NormSpec, y):
        check(lib().bch_matvec_swiglu(self.handle, int(fmt), _view(gate), _view(up), n_rows, n_cols,
                                      _view(x), norm.c(), _view(y)))

    def matvec_conv(self, fmt, weights, n_cols, x, norm: NormSpec | None, taps, history, out,
                    n_embd, kernel_size):
        n = C.byref(norm.c()) if norm is not None else None
        check(lib().bch_matvec_conv(self.handle, int(fmt), _view(weights), n_cols, _view(x), n,
                                    _view(taps), _view(history), _view(out), n_embd, kernel_size))

    def short_conv(self, bcx, taps, history, out, n_embd, kernel_size, n_tokens):
        check(lib().bch_short_conv(self.handle, _view(bcx), _view(taps), _view(history), _view(out),
                                   n_embd, kernel_size, n_tokens))

    def short_conv_batch(self, bcx, taps, history, out, n_embd, kernel_size, n_tokens):
        check(lib().bch_short_conv_batch(self.handle, _view(bcx), _view(taps), _view(history),
                                         _view(out), n_embd, kernel_size, n_tokens))

    def rms_norm(self, x, weight, out, n, n_rows, eps):
        check(lib().bch_rms_norm(self.handle, _view(x), _view(weight), _view(out), n, n_rows, eps))

    def norm_rope(self, src, dst, dst_half, weight, n_heads, head_dim, n_rot, src_head_stride, pos,
                  n_tokens, src_stride, dst_stride, theta, eps):
        check(lib().bch_norm_rope(self.handle, _view(src), _view(dst), int(dst_half), _view(weight),
                                  n_heads, head_dim, n_rot, src_head_stride, pos, n_tokens,
                                  src_stride, dst_stride, theta, eps))

    def convert_half(self, src, dst, n):
        check(lib().bch_convert_half(self.handle, _view(src), _view(dst), n))

    def copy(self, src, dst, n):
        check(lib().bch_copy(self.handle, _view(src), _view(dst), n))

    def embed(self, fmt, weights, n_vocab, tokens, out, n_embd, n_tokens):
        check(lib().bch_embed(self.handle, int(fmt), _view(weights), n_vocab, _view(tokens),
                              _view(out), n_embd, n_tokens))

    def attention(self, q, k_cache, v_cache, kv_half, scratch, out, n_heads, n_kv_heads, head_dim,
                  first_pos, n_queries, n_ctx):
        check(lib().bch_attention(self.handle, _view(q), _view(k_cache), _view(v_cache), int(kv_half),
                                  _view(scratch), _view(out), n_heads, n_kv_heads, head_dim,
                                  first_pos, n_queries, n_ctx))

    def attention_prefill(self, q, k_cache, v_cache, out, n_heads, n_kv_heads, head_dim, first_pos, n_queries,
                          n_ctx):
        check(lib().bch_attention_prefill(self.handle, _view(q), _view(k_cache), _view(v_cache), _view(out),
                                          n_heads, n_kv_heads, head_dim, first_pos, n_queries, n_ctx))

    def attention_decode(self, q, k, v, q_norm, k_norm, eps, rope_theta, n_rot, k_cache, v_cache, kv_half, scratch,
                         out, n_heads, n_kv_heads, head_dim, pos, n_ctx):
        check(lib().bch_attention_decode(self.handle, _view(q), _view(k), _view(v), _view(q_norm), _view(k_norm),
                                         eps, rope_theta, n_rot, _view(k_cache), _view(v_cache), int(kv_half),
                                         _view(scratch), _view(out), n_heads, n_kv_heads, head_dim, pos, n_ctx))

    def kv_plan(self, fmt, n_kv_heads, head_dim, page_size, n_pages, n_heads) -> KvPlan:
        return KvPlan(self, kv_shape(fmt, n_kv_heads, head_dim, page_size, n_pages), n_heads)

    def kv_store(self, plan: KvPlan, cache, k, k_stride, v, v_stride):
        check(lib().bch_kv_store(self.handle, plan.handle, _view(cache), _view(k), k_stride, _view(v), v_stride))

    def kv_load(self, plan: KvPlan, cache, seq, first, n, k, v):
        check(lib().bch_kv_load(self.handle, plan.handle, _view(cache), seq, first, n, _view(k), _view(v)))

    def attention_paged(self, plan: KvPlan, cache, q, q_stride, out, out_stride):
        check(lib().bch_attention_paged(self.handle, plan.handle, _view(cache), _view(q), q_stride, _view(out),
                                        out_stride))

    def logits_edit(self, logits, out, n_rows, n_vocab, rows, *, history=None, n_history=0, bias_tokens=None,
                    bias_values=None, n_bias=0, masks=None, n_masks=0):
        """`rows` holds n_rows LOGIT_ROW; a list of no entries needs no view."""
        view = lambda v: _View() if v is None else _view(v)  # noqa: E731
        rules = LogitRules(view(rows), view(history), view(bias_tokens), view(bias_values), view(masks), n_history,
                           n_bias, n_masks)
        check(lib().bch_logits_edit(self.handle, _view(logits), _view(out), n_rows, n_vocab, C.byref(rules)))

    def matmul(self, fmt, weights, n_rows, n_cols, x, y, n_tokens, store: Store):
        check(lib().bch_matmul(self.handle, int(fmt), _view(weights), n_rows, n_cols, _view(x),
                               _view(y), n_tokens, int(store)))

    def read_sum(self, src, n_vectors, out, n_threads):
        check(lib().bch_read_sum(self.handle, _view(src), n_vectors, _view(out), n_threads))

    def moe_route(self, x, norm: NormSpec | None, normed, router, bias, route, n_cols, n_experts, n_used,
                  n_tokens):
        n = C.byref(norm.c()) if norm is not None else None
        check(lib().bch_moe_route(self.handle, _view(x), n, _view(normed if normed is not None else x),
                                  _view(router), _view(bias), _view(route), n_cols, n_experts, n_used, n_tokens))

    def matvec_experts_swiglu(self, fmt, gate, up, n_rows, n_cols, n_experts, x, route, n_used, y, n_tokens):
        check(lib().bch_matvec_experts_swiglu(self.handle, int(fmt), _view(gate), _view(up), n_rows, n_cols,
                                              n_experts, _view(x), _view(route), n_used, _view(y), n_tokens))

    def matvec_experts_down(self, fmt, weights, n_rows, n_cols, n_experts, x, route, n_used, y, n_tokens):
        check(lib().bch_matvec_experts_down(self.handle, int(fmt), _view(weights), n_rows, n_cols, n_experts,
                                            _view(x), _view(route), n_used, _view(y), n_tokens))

    def moe_group(self, route, offsets, entries, n_experts, n_used, n_tokens):
        check(lib().bch_moe_group(self.handle, _view(route), _view(offsets), _view(entries), n_experts, n_used,
                                  n_tokens))

    def matmul_experts(self, fmt, weights, up, n_rows, n_cols, n_experts, x, shared_input, offsets, entries,
                       n_used, y, n_tokens):
        upv = C.byref(_view(up)) if up is not None else None
        check(lib().bch_matmul_experts(self.handle, int(fmt), _view(weights), upv, n_rows, n_cols, n_experts,
                                       _view(x), int(bool(shared_input)), _view(offsets), _view(entries), n_used,
                                       _view(y), n_tokens))

    def moe_combine(self, x, route, y, n_embd, n_used, n_tokens):
        check(lib().bch_moe_combine(self.handle, _view(x), _view(route), _view(y), n_embd, n_used, n_tokens))

    def sample(self, logits, n_vocab, recent, n_recent, settings, rng_state, out):
        check(lib().bch_sample(self.handle, _view(logits), n_vocab, _view(recent), n_recent, C.byref(settings),
                               _view(rng_state), _view(out)))

    def sample_draw(self, logits, n_vocab, recent, n_recent, settings, u, out):
        check(lib().bch_sample_draw(self.handle, _view(logits), n_vocab, _view(recent), n_recent, C.byref(settings),
                                    u, _view(out)))

    def argmax(self, x, out, n):
        check(lib().bch_argmax(self.handle, _view(x), _view(out), n))


def attention_scratch_floats(n_heads: int, head_dim: int, n_ctx: int, n_queries: int) -> int:
    return lib().bch_attention_scratch_floats(n_heads, head_dim, n_ctx, n_queries)


def attention_decode_scratch_floats(n_heads: int, head_dim: int, n_ctx: int, kv_half: bool) -> int:
    return lib().bch_attention_decode_scratch_floats(n_heads, head_dim, n_ctx, int(kv_half))


def row_bytes(fmt: int, n_cols: int) -> int:
    return lib().bch_row_bytes(int(fmt), n_cols)


__all__ = ["Hip", "Buffer", "KvFormat", "KvPlan", "LOGIT_ROW", "NO_MASK", "ViewRef", "NormSpec", "Format", "Store",
           "BobcatError", "attention_scratch_floats", "attention_decode_scratch_floats", "kv_page_bytes",
           "kv_plan_check", "kv_shape", "row_bytes"]
