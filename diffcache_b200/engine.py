"""Host-side mirror of the reference engine class ``DiffCacheCPU``.

Same constructor, method names, argument meaning and error behaviour as the pyo3
class in diffcache_cpu/src/lib.rs:523-660, with the work done by the CUDA engine
behind the C ABI.  bf16 data crosses as ``uint16`` bit patterns exactly like the
reference (src/diffcache/kvcache/diffcache.py:81-84); every array argument may be
a numpy array (host) or a torch tensor (host or CUDA).
"""
from __future__ import annotations

import ctypes
import functools
import time
from typing import Optional, Sequence

import numpy as np

from . import _lib

BF16, FP16 = 0, 1

_OPTION_DEFAULTS = dict(  # diffcache_cpu/src/lib.rs:556-566
    max_ctx_len=1000000,
    m=16,
    ef_cons=200,
    r_sq=None,
    batch_search=False,
    name="l0",
    use_bruteforce=False,
    attn_mass_threshold=0.9,
    k_check_seq=[100, 200, 300, 400, 800, 1600, 3200, 6400, 12800, 25600],
)


def init_metrics() -> None:
    """Counterpart of ``diffcache._cpu.init_metrics`` (lib.rs:662-665).

    The reference installs a TCP exporter for its per-layer latency counters; this
    engine keeps the same counters, under the reference's names, in
    ``DiffCacheGPU.metrics`` instead, so there is nothing to install."""
    return None


def _metric_names(name: str) -> dict:
    """The reference's counters (microseconds for the latencies): ``{name}_num_searches`` and
    ``{name}_search_latency`` per (batch, kv-head) search (nsw.rs:595,618), ``{name}_collect_latency``
    (nsw.rs:660), ``{name}_total_query_latency`` per query call (lib.rs:403); ``{name}_num_queries``
    counts the calls."""
    return {f"{name}_{k}": 0 for k in ("num_queries", "num_searches", "search_latency", "collect_latency",
                                       "total_query_latency")}


def _is_torch(x) -> bool:
    return type(x).__module__.startswith("torch")


def _ptr(x) -> Optional[int]:
    if x is None:
        return None
    if isinstance(x, np.ndarray):
        return x.ctypes.data
    if _is_torch(x):
        return x.data_ptr()
    if isinstance(x, int):
        return x
    raise TypeError(f"unsupported buffer type {type(x)}")


def _shape(x):
    return tuple(x.shape)


def _require_contiguous(x, what: str) -> None:
    ok = x.flags["C_CONTIGUOUS"] if isinstance(x, np.ndarray) else x.is_contiguous()
    if not ok:
        # the reference reshapes with into_shape_with_order(...).unwrap(), lib.rs:384-385
        raise ValueError(f"{what} must be C-contiguous")


def _require_u16(x, what: str) -> None:
    if isinstance(x, np.ndarray):
        if x.dtype != np.uint16:
            raise TypeError(f"{what}: expected uint16 bit patterns, got {x.dtype}")
    elif x.element_size() != 2:
        raise TypeError(f"{what}: expected a 16-bit element type, got {x.dtype}")


def _current_stream(stream) -> int:
    if stream is not None:
        return int(stream)
    import torch

    return int(torch.cuda.current_stream().cuda_stream)


@functools.lru_cache(maxsize=None)
def _element_types():
    import torch

    return {BF16: (torch.bfloat16, torch.uint16, torch.int16), FP16: (torch.float16, torch.uint16, torch.int16)}


@functools.lru_cache(maxsize=None)
def _word_types(floats: bool):
    import torch

    return (torch.float32,) if floats else (torch.int32, torch.uint32)


@functools.lru_cache(maxsize=None)
def _raw_stream_getter():
    import torch

    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # a tenth of the time of building a Stream object
    return raw if raw is not None else lambda device: torch.cuda.current_stream(device).cuda_stream


def _device_stream(device: int) -> int:
    return int(_raw_stream_getter()(device))


def _alike(x, y) -> bool:
    """Two tensors of one shape, type, device and layout: what holds for one holds for the other."""
    return (type(x) is type(y) and _is_torch(x) and x.shape == y.shape and x.dtype is y.dtype and
            x.get_device() == y.get_device() and x.stride() == y.stride())


def _row_strides(x, what: str):
    """Element strides of the (batch, head, row) axes; 0 for an axis of size 1, whose stride is never used."""
    if isinstance(x, np.ndarray):
        st = tuple(s // x.itemsize for s in x.strides)
    else:
        st = x.stride()
    shp = x.shape
    if st[3] != 1 and shp[3] > 1:
        raise ValueError(f"{what}: head_dim axis must be contiguous")
    return (st[0] if shp[0] != 1 else 0, st[1] if shp[1] != 1 else 0, st[2] if shp[2] != 1 else 0)


class DiffCacheGPU:
    """``DiffCacheCPU(bsz, q_head_num, kv_head_num, head_dim, **kwargs)`` on a B200.

    Accepted kwargs are exactly the reference's (lib.rs:567-582): ``max_ctx_len, m,
    ef_cons, r_sq, batch_search, name, use_bruteforce, attn_mass_threshold,
    k_check_seq``; any other key raises (the reference panics with "Unknown option").
    The graph parameters are accepted and ignored: this engine always runs the exact
    scan, i.e. the reference's ``use_bruteforce=True`` semantics.  Two keyword-only
    additions select the element type and device: ``dtype`` ("bf16" | "fp16") and
    ``device`` (CUDA ordinal); ``adaptive_budget=True`` applies the reference's k-check
    (``k_check_seq``, ``attn_mass_threshold``) to the fused step.  ``store_bits=4`` holds the
    rows in 4 bits (groups of 32 elements with one scale, see ``dc_create_q4``): every method
    works on the rows as they are read back, the store is 3.56 times smaller and the scan reads
    that much less."""

    def __init__(self, bsz: int, q_head_num: int, kv_head_num: int, head_dim: int, **kwargs):
        dtype = kwargs.pop("dtype", "bf16")
        device = kwargs.pop("device", None)
        store_bits = kwargs.pop("store_bits", 16)
        adaptive = bool(kwargs.pop("adaptive_budget", False))
        opts = dict(_OPTION_DEFAULTS)
        for key, value in kwargs.items():
            if key not in opts:
                raise ValueError(f"Unknown option {key}")
            opts[key] = value
        if store_bits not in (4, 16):
            raise ValueError(f"store_bits must be 4 or 16, got {store_bits}")
        self.store_bits = int(store_bits)
        if opts["r_sq"] is None:
            opts["r_sq"] = [4.0] * kv_head_num
        self.options = opts
        self.bsz, self.q_head_num, self.kv_head_num, self.head_dim = bsz, q_head_num, kv_head_num, head_dim
        self.dtype = {"bf16": BF16, "fp16": FP16, BF16: BF16, FP16: FP16}[dtype]
        if device is None:
            import torch

            device = torch.cuda.current_device()
        self.device = int(device)
        self.name = opts["name"]
        self.metrics = _metric_names(self.name)
        self._lib = _lib.load()
        handle = ctypes.c_void_p()
        create = self._lib.dc_create_q4 if self.store_bits == 4 else self._lib.dc_create
        _lib.check(create(bsz, q_head_num, kv_head_num, head_dim, int(opts["max_ctx_len"]), self.dtype,
                          self.device, ctypes.byref(handle)))
        self._h = handle
        if adaptive:
            self.set_adaptive_budget(opts["k_check_seq"], opts["attn_mass_threshold"])

    # -- lifetime ------------------------------------------------------------------------
    def close(self) -> None:
        h, self._h = getattr(self, "_h", None), None
        if h:
            self._lib.dc_destroy(h)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def ctx_len(self) -> int:
        out = ctypes.c_int64()
        _lib.check(self._lib.dc_ctx_len(self._h, ctypes.byref(out)))
        return out.value

    @property
    def group(self) -> int:
        return self.q_head_num // self.kv_head_num

    # -- reference API ---------------------------------------------------------------------
    def prefill(self, keys, vals, neighbours=None, stream=None) -> None:
        """lib.rs:601-611.  keys/vals ``(bsz, kv_head_num, seq_len, head_dim)`` uint16
        (any strides whose last axis is contiguous); ``neighbours`` is accepted and
        ignored (it only feeds the reference's NSW graph)."""
        _require_u16(keys, "keys")
        _require_u16(vals, "vals")
        shp = _shape(keys)
        if len(shp) != 4 or shp[0] != self.bsz or shp[1] != self.kv_head_num or shp[3] != self.head_dim:
            raise ValueError(f"keys shape {shp} != (bsz, kv_head_num, seq_len, head_dim)")
        if _shape(vals) != shp:
            raise ValueError(f"vals shape {_shape(vals)} != keys shape {shp}")

        def strides(x):
            if isinstance(x, np.ndarray):
                st = tuple(s // x.itemsize for s in x.strides)
            else:
                st = tuple(x.stride())
            if st[3] != 1 and shp[3] > 1:
                raise ValueError("head_dim axis must be contiguous")
            return st

        sk, sv = strides(keys), strides(vals)
        if sk != sv:
            raise ValueError("keys and vals must share one stride pattern")
        _lib.check(self._lib.dc_prefill(self._h, _ptr(keys), _ptr(vals), shp[2], sk[0], sk[1], sk[2],
                                        _current_stream(stream)))

    def insert(self, keys, vals, stream=None) -> None:
        """lib.rs:591-599.  keys/vals ``(bsz, kv_head_num, head_dim)``."""
        for x, what in ((keys, "keys"), (vals, "vals")):
            _require_u16(x, what)
            _require_contiguous(x, what)
            if _shape(x) != (self.bsz, self.kv_head_num, self.head_dim):
                raise ValueError(f"{what} shape {_shape(x)} != (bsz, kv_head_num, head_dim)")
        _lib.check(self._lib.dc_insert(self._h, _ptr(keys), _ptr(vals), _current_stream(stream)))

    def query(self, out_keys, out_vals, queries, ef: int, out_idx=None, out_bits=None, stream=None) -> None:
        """lib.rs:613-624 with ``use_bruteforce`` semantics (nsw.rs:592-630).

        ``queries`` ``(bsz, kv_head_num, head_dim)``; ``out_keys/out_vals``
        ``(bsz, kv_head_num, min(ef, ctx_len), head_dim)`` C-contiguous; row ``i`` is the
        ``i``-th best key.  ``out_idx`` (int32) / ``out_bits`` (uint32) optionally receive the
        selected row ids and their ranking keys."""
        _require_u16(queries, "queries")
        _require_contiguous(queries, "queries")
        if _shape(queries) != (self.bsz, self.kv_head_num, self.head_dim):
            raise ValueError(f"queries shape {_shape(queries)} != (bsz, kv_head_num, head_dim)")
        ef_c = min(int(ef), self.ctx_len)
        for x, what in ((out_keys, "out_keys"), (out_vals, "out_vals")):
            if x is None:
                continue
            _require_u16(x, what)
            _require_contiguous(x, what)
            if _shape(x) != (self.bsz, self.kv_head_num, ef_c, self.head_dim):
                raise ValueError(f"{what} shape {_shape(x)} != (bsz, kv_head_num, {ef_c}, head_dim)")
        for x, what in ((out_idx, "out_idx"), (out_bits, "out_bits")):
            if x is not None:
                _require_contiguous(x, what)
                if _shape(x) != (self.bsz, self.kv_head_num, ef_c):
                    raise ValueError(f"{what} shape {_shape(x)} != (bsz, kv_head_num, {ef_c})")
        t0 = time.perf_counter()
        _lib.check(self._lib.dc_query(self._h, _ptr(queries), int(ef), _ptr(out_keys), _ptr(out_vals), _ptr(out_idx),
                                      _ptr(out_bits), _current_stream(stream)))
        # wall time of the call, as the reference measures it (lib.rs:378,403); with device outputs the call only
        # enqueues work, so device time has to come from set_phase_timing / phase_times
        self._count_query(int((time.perf_counter() - t0) * 1e6))

    def query_streaming(self, cuda_stream: int, out_keys_gpu: int, out_vals_gpu: int, queries, ef: int) -> None:
        """lib.rs:626-636: raw ``CUstream`` / device pointers as integers.  The reference
        streams chunks as its graph search converges; an exact scan has a single final
        answer, so this writes the complete result to the device buffers on ``cuda_stream``."""
        _require_u16(queries, "queries")
        _lib.check(self._lib.dc_query(self._h, _ptr(queries), int(ef), int(out_keys_gpu), int(out_vals_gpu), None, None,
                                      int(cuda_stream)))

    def _count_query(self, total_us: int = 0) -> None:
        m, n = self.metrics, self.name
        m[f"{n}_num_queries"] += 1
        m[f"{n}_num_searches"] += self.bsz * self.kv_head_num   # one search per (batch, kv head), nsw.rs:595
        m[f"{n}_total_query_latency"] += total_us

    def get_keys(self) -> np.ndarray:
        """lib.rs:646-649: stored keys as float32 ``(bsz, kv_head_num, ctx_len, head_dim)``."""
        out = np.empty((self.bsz, self.kv_head_num, self.ctx_len, self.head_dim), np.float32)
        _lib.check(self._lib.dc_get_keys(self._h, out.ctypes.data))
        return out

    def update_r_sq(self, r_sq: Sequence[float]) -> None:
        """lib.rs:651-659: validated and otherwise unused (r_sq never enters QKDist)."""
        arr = np.asarray(list(r_sq), np.float32)
        _lib.check(self._lib.dc_update_r_sq(self._h, arr.ctypes.data, int(arr.shape[0])))
        self.options["r_sq"] = [float(x) for x in arr]

    def save(self, path: str) -> None:
        """lib.rs:638-640.  Snapshot format: see :mod:`diffcache_b200.snapshot`."""
        from . import snapshot

        snapshot.save_engine(self, path)

    def load(self, path: str, ctx_len: int) -> None:
        """lib.rs:642-644."""
        from . import snapshot

        snapshot.load_engine(self, path, ctx_len)

    # -- stored rows -------------------------------------------------------------------------
    def write_rows(self, row0: int, keys, vals, stream=None) -> None:
        """Writes (or overwrites) stored rows ``[row0, row0 + n)``, e.g. one chunk of a chunked prefill;
        ``keys``/``vals`` ``(bsz, kv_head_num, n, head_dim)`` as in :meth:`prefill`.  ``row0`` may be at most
        ``ctx_len``; the store then holds ``max(ctx_len, row0 + n)`` rows."""
        n = self._rows(keys, None, "keys")
        sb, sh, ss = _row_strides(keys, "keys")
        if not _alike(keys, vals):
            self._rows(vals, n, "vals")
            if _row_strides(vals, "vals") != (sb, sh, ss):
                raise ValueError("keys and vals must share one stride pattern")
        _lib.check(self._lib.dc_write_rows(self._h, _ptr(keys), _ptr(vals), int(row0), n, sb, sh, ss, self._stream(stream)))

    def read_rows(self, out_keys, out_vals, row0: int = 0, ids=None, stream=None) -> None:
        """Reads stored rows back into ``out_keys``/``out_vals`` ``(bsz, kv_head_num, n, head_dim)`` (dense device
        tensors of the element type; ``None`` skips one): rows ``row0 ..``, or the rows ``ids`` ``(bsz,
        kv_head_num, n)`` int32.  Rows that are not stored (negative ids, positions beyond ``ctx_len``) are zeros."""
        n = None
        for x, what in ((out_keys, "out_keys"), (out_vals, "out_vals")):
            if x is not None and not (n is not None and _alike(out_keys, x)):
                self._on_device(x, what)
                n = self._rows(x, n, what)
                _require_contiguous(x, what)
        if n is None:
            return
        if ids is not None:
            self._words(ids, (self.bsz, self.kv_head_num, n), "ids")
        _lib.check(self._lib.dc_read_rows(self._h, int(row0), _ptr(ids), n, _ptr(out_keys), _ptr(out_vals),
                                          self._stream(stream)))

    def score_rows(self, q, out_bits, stream=None) -> None:
        """Ranking keys ``bits(65536 - <q, k>)`` of the first ``n`` stored rows into ``out_bits`` ``(bsz, kv_head_num,
        n)`` (32-bit device tensor; entries beyond the stored rows stay as they are).  ``q`` ``(bsz, kv_head_num,
        head_dim)`` holds one (group-mean) vector per kv head, or ``(bsz, q_head_num, head_dim)`` the query
        heads, whose group mean is taken."""
        mode = 0 if len(q.shape) == 3 and q.shape[1] == self.kv_head_num else 1
        self._heads(q, self.kv_head_num if mode == 0 else self.q_head_num, "q")
        _require_contiguous(q, "q")
        n = self._words(out_bits, (self.bsz, self.kv_head_num, None), "out_bits")
        _lib.check(self._lib.dc_score_rows(self._h, q.data_ptr(), mode, n, out_bits.data_ptr(), n, self._stream(stream)))

    def attend_rows(self, q, out, ids=None, lens=None, res_k=None, res_v=None, res_len: int = 0, k_new=None, v_new=None,
                    scale: float = 0.0, out_lse=None, stream=None) -> None:
        """Softmax attention of every query head over the stored rows ``ids`` ``(bsz, kv_head_num, k)`` int32 (ids that
        are not stored are skipped), the resident rows and the new token; arguments as in :meth:`decode_attend`.
        Without ``ids`` (4-bit stores): every stored row, of sequence ``b`` only the first ``lens[b]`` (int32
        device tensor ``(bsz,)``) when ``lens`` is given.  Heads that have nothing to attend over get 0, and -inf in
        ``out_lse`` ``(bsz, q_head_num)`` float32.  Calls of one engine share its scratch: order them."""
        self._heads(q, self.q_head_num, "q")
        self._heads(out, self.q_head_num, "out")
        _require_contiguous(out, "out")
        qsb = 0 if q.is_contiguous() else self._slice_stride(q, self.q_head_num, "q")
        n_ids, ids_ptr, lens_ptr, lse_ptr, kn_ptr, vn_ptr, nsb, rk_ptr, rv_ptr, sb, sh = -1, None, None, None, None, None, 0, None, None, 0, 0
        if ids is not None:
            if lens is not None:
                raise ValueError("lens only limits attention over all rows: give ids or lens")
            n_ids = self._words(ids, (self.bsz, self.kv_head_num, None), "ids")
            ids_ptr = ids.data_ptr() if n_ids > 0 else None
        elif self.store_bits != 4:
            raise ValueError("attention over every stored row needs store_bits=4; give ids")
        elif lens is not None:
            self._words(lens, (self.bsz,), "lens")
            lens_ptr = lens.data_ptr()
        if out_lse is not None:
            self._words(out_lse, (self.bsz, self.q_head_num), "out_lse")
            lse_ptr = out_lse.data_ptr()
        if (k_new is None) != (v_new is None) or (res_k is None) != (res_v is None):
            raise ValueError("k_new and v_new, res_k and res_v come in pairs")
        need = int(res_len)
        if need < 0:
            raise ValueError("res_len must not be negative")
        if k_new is not None:
            self._heads(k_new, self.kv_head_num, "k_new")
            self._heads(v_new, self.kv_head_num, "v_new")
            if not (k_new.is_contiguous() and v_new.is_contiguous()):
                nsb = self._slice_stride(k_new, self.kv_head_num, "k_new")
                if self._slice_stride(v_new, self.kv_head_num, "v_new") != nsb:
                    raise ValueError("k_new and v_new must have the same batch stride")
            kn_ptr, vn_ptr = k_new.data_ptr(), v_new.data_ptr()
            need += 1
        if res_k is not None:
            self._on_device(res_k, "res_k")
            rows = self._rows(res_k, None, "res_k")
            sb, sh, ss = _row_strides(res_k, "res_k")
            if not _alike(res_k, res_v):
                self._on_device(res_v, "res_v")
                self._rows(res_v, rows, "res_v")
                if (sb, sh, ss) != _row_strides(res_v, "res_v"):
                    raise ValueError("res_k/res_v must share strides with contiguous rows of head_dim")
            if rows < need:
                raise ValueError(f"res_k/res_v hold {rows} rows, the call needs {need}")
            if ss not in (0, self.head_dim):
                raise ValueError("res_k/res_v must share strides with contiguous rows of head_dim")
            rk_ptr, rv_ptr = res_k.data_ptr(), res_v.data_ptr()
        elif res_len:
            raise ValueError("res_len > 0 needs res_k and res_v")
        _lib.check(self._lib.dc_attend_rows(self._h, q.data_ptr(), qsb, ids_ptr, n_ids, lens_ptr, kn_ptr, vn_ptr, nsb, rk_ptr, rv_ptr,
                                            sb, sh, int(res_len), float(scale), out.data_ptr(), lse_ptr, self._stream(stream)))

    # Argument checks of the calls above.  They are the larger part of a small call's time, so each looks at an
    # attribute once.
    def _stream(self, stream) -> int:
        """The given stream, else the current stream of this engine's device."""
        return _device_stream(self.device) if stream is None else int(stream)

    def _slice_stride(self, x, heads: int, what: str) -> int:
        if self.bsz > 1 and x.stride(0) == 0:   # 0 means dense to the engine
            raise ValueError(f"{what} must not be expanded over the batch")
        return self._batch_stride(x, heads, what)

    def _on_device(self, x, what: str) -> None:
        if not _is_torch(x):
            raise TypeError(f"{what} must be a device tensor, got {type(x)}")
        if x.get_device() != self.device:   # -1 for host tensors
            raise ValueError(f"{what} must be a device tensor on cuda:{self.device}, got one on {x.device}")

    def _rows(self, x, n, what: str) -> int:
        """Rows (bsz, kv_head_num, n, head_dim) of the element type or its 16-bit patterns, in host memory or on this
        engine's device; n None: any.  Returns n."""
        if _is_torch(x):
            if x.dtype not in _element_types()[self.dtype]:
                raise TypeError(f"{what}: expected {_element_types()[self.dtype][0]} or 16-bit patterns, got {x.dtype}")
            if x.get_device() not in (-1, self.device):
                raise ValueError(f"{what} is on {x.device}, the engine on cuda:{self.device}")
        else:
            _require_u16(x, what)
        shape = x.shape
        if len(shape) != 4 or shape[0] != self.bsz or shape[1] != self.kv_head_num or shape[3] != self.head_dim or n not in (None, shape[2]):
            raise ValueError(f"{what} shape {tuple(shape)} != {(self.bsz, self.kv_head_num, 'any' if n is None else n, self.head_dim)}")
        return shape[2]

    def _heads(self, x, heads: int, what: str) -> None:
        """(bsz, heads, head_dim) of the element type on this engine's device."""
        self._on_device(x, what)
        if x.dtype not in _element_types()[self.dtype]:
            raise TypeError(f"{what}: expected {_element_types()[self.dtype][0]} or 16-bit patterns, got {x.dtype}")
        if x.shape != (self.bsz, heads, self.head_dim):
            raise ValueError(f"{what} shape {tuple(x.shape)} != {(self.bsz, heads, self.head_dim)}")

    def _words(self, x, shape, what: str) -> int:
        """A dense 32-bit tensor of this shape (last size None: any) on this engine's device; returns its last size."""
        self._on_device(x, what)
        if x.dtype not in _word_types(what == "out_lse"):
            raise TypeError(f"{what}: expected one of {_word_types(what == 'out_lse')}, got {x.dtype}")
        got = tuple(x.shape)
        if got != shape and (shape[-1] is not None or len(got) != len(shape) or got[:-1] != shape[:-1]):
            raise ValueError(f"{what} shape {got} != {tuple('any' if w is None else w for w in shape)}")
        if not x.is_contiguous():
            raise ValueError(f"{what} must be C-contiguous")
        return got[-1]

    # -- fused device path -----------------------------------------------------------------
    def set_row_offset(self, row_offset: int) -> None:
        _lib.check(self._lib.dc_set_row_offset(self._h, int(row_offset)))

    def check_status(self, stream=None) -> None:
        _lib.check(self._lib.dc_check_status(self._h, _current_stream(stream)))

    def decode_attend(self, q, out, topk: int, res_k=None, res_v=None, res_len: int = 0, k_new=None, v_new=None,
                      scale: float = 0.0, out_idx=None, out_lse=None, stream=None) -> None:
        """One fused decode step on device tensors (see ``dc_decode_attend``).

        ``q``/``out`` ``(bsz, q_head_num, head_dim)``; ``res_k/res_v`` a view
        ``(bsz, kv_head_num, rows, head_dim)`` of the resident sink+window buffer whose first
        ``res_len`` rows are valid; ``k_new/v_new`` ``(bsz, kv_head_num, head_dim)``.  ``q``, ``k_new`` and
        ``v_new`` may be slices of a fused projection output: heads dense inside a batch, any batch stride
        (``k_new`` and ``v_new`` the same one)."""
        qsb = self._batch_stride(q, self.q_head_num, "q")
        nsb = 0
        if k_new is not None:
            nsb = self._batch_stride(k_new, self.kv_head_num, "k_new")
            if self._batch_stride(v_new, self.kv_head_num, "v_new") != nsb:
                raise ValueError("k_new and v_new must have the same batch stride")
        sb = sh = 0
        if res_k is not None:
            st = tuple(res_k.stride())
            if st != tuple(res_v.stride()) or st[3] != 1 or st[2] != self.head_dim:
                raise ValueError("res_k/res_v must share strides with contiguous rows of head_dim")
            sb, sh = st[0], st[1]
        _lib.check(self._lib.dc_decode_attend_strided(self._h, _ptr(q), qsb, _ptr(k_new), _ptr(v_new), nsb, _ptr(res_k),
                                                      _ptr(res_v), sb, sh, int(res_len), int(topk), float(scale),
                                                      _ptr(out), _ptr(out_idx), _ptr(out_lse), _current_stream(stream)))
        self._count_query()

    def set_output_exchange(self, exchange, channel: int = 0) -> None:
        """Head-sharded layers: every following ``decode_attend*`` call also stores its output slice into every
        rank's copy of ``channel`` of ``exchange`` (a :class:`diffcache_b200.sharded.PeerExchange`; ``None``
        switches it off), interleaved so that the channel reads ``(bsz, world, q_head_num * head_dim)``."""
        _lib.check(self._lib.dc_set_output_exchange(self._h, None if exchange is None else exchange._h, int(channel)))

    def set_output_gather(self, dense) -> None:
        """After :meth:`set_output_exchange`: the kernel that stores the slice also waits for every rank's slice
        and writes all of them to ``dense`` ``(bsz, world * q_head_num * head_dim)`` (a device tensor that must
        stay alive; ``None`` switches it off), so no separate ``PeerExchange.collect`` is needed.  Ranks must
        run on different GPUs."""
        _lib.check(self._lib.dc_set_output_gather(self._h, _ptr(dense)))
        self._out_dense = dense

    def window_push(self, k_new, v_new, res_k, res_v, window_state, stream=None) -> None:
        """Append the step's new token to this layer's window ring (see ``dc_window_push``): the oldest
        token is spilled into the scanned store once the window is full.  ``window_state`` is the int32
        device tensor of 8 words shared by all layers."""
        nsb = self._batch_stride(k_new, self.kv_head_num, "k_new")
        if self._batch_stride(v_new, self.kv_head_num, "v_new") != nsb:
            raise ValueError("k_new and v_new must have the same batch stride")
        st = tuple(res_k.stride())
        if st != tuple(res_v.stride()) or st[3] != 1 or st[2] != self.head_dim:
            raise ValueError("res_k/res_v must share strides with contiguous rows of head_dim")
        _lib.check(self._lib.dc_window_push(self._h, _ptr(k_new), _ptr(v_new), nsb, _ptr(res_k), _ptr(res_v), st[0], st[1],
                                            _ptr(window_state), _current_stream(stream)))

    def window_advance(self, window_state, stream=None) -> None:
        """Once per decode step, after the last layer's ``window_push``."""
        _lib.check(self._lib.dc_window_advance(_ptr(window_state), _current_stream(stream)))

    def decode_attend_dyn(self, q, out, topk: int, res_k, res_v, res_len_dev, res_cap: int, scale: float = 0.0,
                          out_idx=None, out_lse=None, stream=None) -> None:
        """``decode_attend`` with the resident length (``res_len_dev``, one int32 on the device) and the
        stored row count read on the device when the kernels run, so a captured graph of this call stays
        valid while the window and the store grow.  The new token must already be in the window."""
        qsb = self._batch_stride(q, self.q_head_num, "q")
        st = tuple(res_k.stride())
        if st != tuple(res_v.stride()) or st[3] != 1 or st[2] != self.head_dim:
            raise ValueError("res_k/res_v must share strides with contiguous rows of head_dim")
        _lib.check(self._lib.dc_decode_attend_dyn(self._h, _ptr(q), qsb, _ptr(res_k), _ptr(res_v), st[0], st[1],
                                                  _ptr(res_len_dev), int(res_cap), int(topk), float(scale), _ptr(out),
                                                  _ptr(out_idx), _ptr(out_lse), _current_stream(stream)))
        self._count_query()

    def _batch_stride(self, t, heads: int, what: str) -> int:
        """0 for a dense ``(bsz, heads, head_dim)`` tensor, else its batch stride in elements."""
        if not hasattr(t, "stride"):   # not a torch tensor: taken as dense
            return 0
        st, shape = tuple(t.stride()), tuple(t.shape)
        # the stride of a dimension of size 1 is never used and may hold anything
        if len(st) != 3 or (shape[2] != 1 and st[2] != 1) or (shape[1] != 1 and st[1] != self.head_dim):
            raise ValueError(f"{what} must be (bsz, {heads}, head_dim) with dense heads; strides {st}")
        return 0 if shape[0] == 1 or st[0] == heads * self.head_dim else int(st[0])

    def set_adaptive_budget(self, k_check_seq, attn_mass_threshold: float) -> None:
        """Switch the k-check on for ``decode_attend`` (``k_check_seq`` empty switches it off): per
        (batch, kv-head) the first checkpoint whose top-h keys already hold ``attn_mass_threshold`` of
        the estimated attention mass becomes the number of retrieved rows attended (nsw.rs:198-300)."""
        seq = np.asarray(sorted(int(x) for x in k_check_seq)[:16], np.int32)
        _lib.check(self._lib.dc_set_adaptive_budget(self._h, seq.ctypes.data if seq.size else None, int(seq.size),
                                                    float(attn_mass_threshold)))

    def last_budget(self) -> np.ndarray:
        """Budgets chosen by the last ``decode_attend`` step, ``(bsz, kv_head_num)`` int32."""
        out = np.zeros((self.bsz, self.kv_head_num), np.int32)
        _lib.check(self._lib.dc_get_budget(self._h, out.ctypes.data, _current_stream(None)))
        return out

    def set_phase_timing(self, max_steps: int) -> None:
        """Record CUDA events around the scan / select / attend phases of the next ``max_steps``
        ``decode_attend`` calls (the counterpart of the reference's per-layer latency counters)."""
        _lib.check(self._lib.dc_set_phase_timing(self._h, int(max_steps)))

    def phase_times(self) -> dict:
        """Summed milliseconds per phase over the recorded steps."""
        a, b, c, n = ctypes.c_float(), ctypes.c_float(), ctypes.c_float(), ctypes.c_int()
        _lib.check(self._lib.dc_get_phase_times(self._h, ctypes.byref(a), ctypes.byref(b), ctypes.byref(c),
                                                ctypes.byref(n)))
        # the device-timed phases under the reference's counter names: search = scan + select (nsw.rs:597-618),
        # collect = gather + attention of the selected rows (nsw.rs:620-629 and the attention that follows)
        m, nm = self.metrics, self.name
        m[f"{nm}_search_latency"] += int((a.value + b.value) * 1e3)
        m[f"{nm}_collect_latency"] += int(c.value * 1e3)
        m[f"{nm}_total_query_latency"] += int((a.value + b.value + c.value) * 1e3)
        return {"steps": n.value, "scan_ms": a.value, "select_ms": b.value, "attend_ms": c.value}

    def local_topk(self, q, topk: int, out_bits, out_gidx, stream=None) -> None:
        _lib.check(self._lib.dc_local_topk(self._h, _ptr(q), int(topk), _ptr(out_bits), _ptr(out_gidx),
                                           _current_stream(stream)))

    def attend_owned(self, q, sel_gidx, n_sel: int, out_acc, out_ml, res_k=None, res_v=None, res_len: int = 0,
                     k_new=None, v_new=None, scale: float = 0.0, stream=None, sel_count=None) -> None:
        sb = sh = 0
        if res_k is not None:
            st = tuple(res_k.stride())
            sb, sh = st[0], st[1]
        _lib.check(self._lib.dc_attend_owned(self._h, _ptr(q), _ptr(sel_gidx), int(n_sel), _ptr(k_new), _ptr(v_new),
                                             _ptr(res_k), _ptr(res_v), sb, sh, int(res_len), float(scale),
                                             _ptr(out_acc), _ptr(out_ml), _ptr(sel_count), _current_stream(stream)))
