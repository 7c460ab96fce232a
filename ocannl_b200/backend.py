"""ctypes binding of libb200.so and a host-side mirror of arrayjit's backend interface.

The classes follow the user-facing signatures of arrayjit/lib/backend_intf.ml:
`Backend.compile` / `link` (:319-336), `routine` (:59-70), `context` (:134-149), device
`await` / `all_work` (:97-126) and the host copies `from_host` / `to_host`
(arrayjit/lib/backends.ml:113-158).  `Context.link` restates `Raise_backend.allocate_delta`
(arrayjit/lib/backends.ml:529-614): nodes of the routine that the parent context does not
hold yet are bump-packed into one new pool, zero-initialised unless the routine zeroes them
itself, and the child context records their {pool, offset}.

Everything that computes goes through the C ABI of include/b200.h; when the library or a
GPU is missing the calls raise — there is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import json
import os
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np

from .low_level import PREC_BYTES, Routine as IrRoutine, Tnode

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libb200.so")

NP_DTYPE = {"byte": np.uint8, "uint16": np.uint16, "int32": np.int32, "uint32": np.uint32,
            "int64": np.int64, "uint64": np.uint64, "half": np.float16, "bfloat16": np.uint16,
            "fp8": np.uint8, "single": np.float32, "double": np.float64,
            # four 32-bit words per element: arrays of this precision get a trailing axis of 4
            "uint4x32": np.dtype((np.uint32, (4,)))}


class B200Error(RuntimeError):
    """Non-zero status from the C ABI; `.code` < 0 is a B200_E_* value, > 0 a CUDA /
    NVRTC / NCCL result."""

    def __init__(self, code: int, msg: str):
        super().__init__("b200 error %d: %s" % (code, msg))
        self.code = code


class UserError(B200Error):
    """Utils.User_error of the reference: bad static index, missing binding."""


class Binding(ctypes.Structure):
    _fields_ = [("tn_id", ctypes.c_int32), ("pool_id", ctypes.c_int32), ("offset", ctypes.c_uint64)]


_lib = None


def lib() -> ctypes.CDLL:
    """Loads libb200.so (built in-tree by `python -m ocannl_b200.build`)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise B200Error(-2, "libb200.so is not built: run `python -m ocannl_b200.build`")
        L = ctypes.CDLL(LIB_PATH)
        L.b200_last_error.restype = ctypes.c_char_p
        L.b200_version.restype = ctypes.c_char_p
        _lib = L
    return _lib


def check(rc: int) -> None:
    if rc != 0:
        msg = lib().b200_last_error().decode(errors="replace")
        raise (UserError if rc == -5 else B200Error)(rc, msg)


def _vp(x) -> ctypes.c_void_p:
    return ctypes.c_void_p(x)


class Event:
    def __init__(self, h):
        self.h = h

    def sync(self):
        check(lib().b200_event_sync(self.h))

    def is_done(self) -> bool:
        d = ctypes.c_int(0)
        check(lib().b200_event_query(self.h, ctypes.byref(d)))
        return bool(d.value)

    def elapsed_ms(self, later: "Event") -> float:
        ms = ctypes.c_float(0)
        check(lib().b200_event_elapsed_ms(self.h, later.h, ctypes.byref(ms)))
        return ms.value

    def free(self):
        if self.h:
            lib().b200_event_free(self.h)
            self.h = None


class Device:
    """One GPU with its stream and pool table (Backend_intf.device)."""

    def __init__(self, ordinal: int = 0):
        h = ctypes.c_void_p()
        check(lib().b200_device_open(ctypes.c_int(ordinal), ctypes.byref(h)))
        self.h = h
        self.ordinal = ordinal
        self._next_pool = 1            # pool id 0 is the merge buffer (backend_intf.ml:131-132)

    def props(self) -> dict:
        buf = ctypes.create_string_buffer(1024)
        check(lib().b200_device_props(self.h, buf, ctypes.c_size_t(1024)))
        return json.loads(buf.value.decode())

    def alloc_pool(self, size_in_bytes: int, pool_id: Optional[int] = None, alignment: int = 256) -> int:
        if pool_id is None:
            pool_id = self._next_pool
            self._next_pool += 1
        check(lib().b200_pool_alloc(self.h, ctypes.c_int(pool_id), ctypes.c_size_t(size_in_bytes),
                                    ctypes.c_size_t(alignment)))
        return pool_id

    def free_pool(self, pool_id: int):
        check(lib().b200_pool_free(self.h, ctypes.c_int(pool_id)))

    def memset_zero(self, pool_id: int, offset: int, size_in_bytes: int):
        check(lib().b200_pool_memset0(self.h, ctypes.c_int(pool_id), ctypes.c_size_t(offset),
                                      ctypes.c_size_t(size_in_bytes)))

    def pool_address(self, pool_id: int) -> Tuple[int, int]:
        p, n = ctypes.c_uint64(0), ctypes.c_size_t(0)
        check(lib().b200_pool_address(self.h, ctypes.c_int(pool_id), ctypes.byref(p), ctypes.byref(n)))
        return p.value, n.value

    def from_host(self, pool_id: int, offset: int, arr: np.ndarray):
        assert arr.flags["C_CONTIGUOUS"]
        check(lib().b200_h2d(self.h, ctypes.c_int(pool_id), ctypes.c_size_t(offset), _vp(arr.ctypes.data),
                             ctypes.c_size_t(arr.nbytes)))

    def to_host(self, pool_id: int, offset: int, arr: np.ndarray):
        assert arr.flags["C_CONTIGUOUS"] and arr.flags["WRITEABLE"]
        check(lib().b200_d2h(self.h, ctypes.c_int(pool_id), ctypes.c_size_t(offset), _vp(arr.ctypes.data),
                             ctypes.c_size_t(arr.nbytes)))

    def device_to_device(self, dst_pool: int, dst_offset: int, src: "Device", src_pool: int, src_offset: int, nbytes: int):
        """Copy between pools of one device or of two (`device_to_device ~into_merge_buffer:No`,
        arrayjit/lib/cuda_backend.ml:289-314), ordered after the work queued on the source."""
        check(lib().b200_d2d(self.h, ctypes.c_int(dst_pool), ctypes.c_size_t(dst_offset), src.h, ctypes.c_int(src_pool),
                             ctypes.c_size_t(src_offset), ctypes.c_size_t(nbytes)))

    def merge_copy(self, src: "Device", src_pool: int, src_offset: int, nbytes: int):
        """`device_to_device ~into_merge_buffer:Copy`: the source node lands in this device's merge
        buffer (pool 0, grown as needed), where a routine's `Get_merge_buffer` reads it."""
        check(lib().b200_merge_copy(self.h, src.h, ctypes.c_int(src_pool), ctypes.c_size_t(src_offset), ctypes.c_size_t(nbytes)))

    def all_work(self) -> Event:
        e = ctypes.c_void_p()
        check(lib().b200_event_record(self.h, ctypes.byref(e)))
        return Event(e)

    def will_wait_for(self, ev: Event):
        check(lib().b200_stream_wait(self.h, ev.h))

    def await_(self):
        check(lib().b200_await(self.h))

    def is_idle(self) -> bool:
        d = ctypes.c_int(0)
        check(lib().b200_is_idle(self.h, ctypes.byref(d)))
        return bool(d.value)

    def set_async_uploads(self, on: bool = True):
        """from_host copies on a second stream (see b200_set_async_uploads in include/b200.h)."""
        check(lib().b200_set_async_uploads(self.h, ctypes.c_int(1 if on else 0)))

    def stream_handle(self) -> int:
        s = ctypes.c_uint64(0)
        check(lib().b200_stream_handle(self.h, ctypes.byref(s)))
        return s.value

    def sum_f32_static(self, in_pool: int, in_offset: int, count: int, out_pool: int, out_offset: int):
        """Sum of `count` floats, written as one float, without any allocation at call time
        (scratch is a fixed 4 KiB array inside the library's device image; count <= 2**26).
        For callers that must not touch the device allocator while running; calls that overlap
        on the GPU share that array and race, stream-ordered calls are safe."""
        check(lib().b200_sum_f32_static(self.h, ctypes.c_int(in_pool), ctypes.c_size_t(in_offset),
                                        ctypes.c_size_t(count), ctypes.c_int(out_pool), ctypes.c_size_t(out_offset)))

    def get_used_memory(self) -> int:
        n = ctypes.c_size_t(0)
        check(lib().b200_used_memory(self.h, ctypes.byref(n)))
        return n.value

    def get_debug_info(self) -> dict:
        buf = ctypes.create_string_buffer(1024)
        check(lib().b200_debug_info(self.h, buf, ctypes.c_size_t(1024)))
        return json.loads(buf.value.decode())


def num_devices() -> int:
    n = ctypes.c_int(0)
    check(lib().b200_num_devices(ctypes.byref(n)))
    return n.value


class PinnedBuffer:
    """Page-locked host memory viewed as a numpy array (for from_host / to_host)."""

    def __init__(self, shape, dtype):
        self.nbytes = int(np.prod(shape)) * np.dtype(dtype).itemsize
        p = ctypes.c_void_p()
        check(lib().b200_host_alloc(ctypes.c_size_t(max(self.nbytes, 1)), ctypes.byref(p)))
        self.ptr = p
        raw = (ctypes.c_char * max(self.nbytes, 1)).from_address(p.value)
        self.array = np.frombuffer(raw, dtype=dtype, count=int(np.prod(shape))).reshape(shape)

    def free(self):
        if self.ptr:
            self.array = None
            lib().b200_host_free(self.ptr)
            self.ptr = None


class Code:
    """Device-independent compiled routine (`Backend.compile`)."""

    def __init__(self, ir: IrRoutine, options: Optional[str] = None, name: Optional[str] = None):
        self.ir = ir
        text = ir.to_b200ir().encode()
        h = ctypes.c_void_p()
        check(lib().b200_compile((name or "").encode(), text, ctypes.c_size_t(len(text)),
                                 options.encode() if options else None, ctypes.byref(h)))
        self.h = h

    def info(self) -> dict:
        buf = ctypes.create_string_buffer(1 << 16)
        check(lib().b200_code_info(self.h, buf, ctypes.c_size_t(1 << 16)))
        return json.loads(buf.value.decode())

    def source(self, stage: int = -1) -> str:
        need = ctypes.c_size_t(0)
        check(lib().b200_code_source(self.h, ctypes.c_int(stage), None, ctypes.c_size_t(0), ctypes.byref(need)))
        buf = ctypes.create_string_buffer(need.value)
        check(lib().b200_code_source(self.h, ctypes.c_int(stage), buf, ctypes.c_size_t(need.value), None))
        return buf.value.decode()

    def free(self):
        if self.h:
            lib().b200_code_free(self.h)
            self.h = None


# ------------------------------------------------------------------ operators
class Operand(ctypes.Structure):
    _fields_ = [("pool_id", ctypes.c_int32), ("offset", ctypes.c_uint64)]


def _spec(name: str, *fields):
    """A struct of include/b200.h; operands that are not set are not given."""
    cls = type(name, (ctypes.Structure,), {"_fields_": [(f, t) for f, t in fields]})

    def init(self, **values):
        ctypes.Structure.__init__(self)
        for f, t in fields:
            if t is Operand:
                setattr(self, f, Operand(-1, 0))
            elif t is Operand * 2:
                setattr(self, f, t(Operand(-1, 0), Operand(-1, 0)))
            elif issubclass(t, ctypes.Structure):
                setattr(self, f, t())
        for k, v in values.items():
            setattr(self, k, v)
    cls.__init__ = init
    return cls


_i32, _i64, _f32 = ctypes.c_int32, ctypes.c_int64, ctypes.c_float
LayerNormSpec = _spec("LayerNormSpec", ("rows", _i64), ("n", _i64), ("dtype", _i32), ("weight_dtype", _i32), ("eps", _f32),
                      *((n, Operand) for n in ("x", "residual", "gamma", "beta", "y", "total", "mean", "rstd", "dy", "d_total", "dx",
                                               "dgamma", "dbeta")))
RotarySpec = _spec("RotarySpec", ("batch", _i64), ("seq", _i64), ("heads", _i32 * 2), ("d", _i32), ("pairs", _i32), ("dtype", _i32),
                   ("interleaved", _i32), ("inverse", _i32), ("magnitude", _f32), ("frequencies", ctypes.POINTER(ctypes.c_double)),
                   ("first_position", _i64), ("positions", Operand), ("x", Operand * 2), ("y", Operand * 2))
AttentionSpec = _spec("AttentionSpec", ("batch", _i64), ("queries", _i64), ("keys", _i64), ("heads", _i32), ("kv_heads", _i32), ("d", _i32),
                      ("dtype", _i32), ("mask", _i32), ("scale", _f32), ("cap", _f32),
                      *((n, Operand) for n in ("q", "k", "v", "out", "lse", "lengths", "prefix", "query_documents", "key_documents",
                                               "slopes", "d_out", "dq", "dk", "dv")))
CacheSpec = _spec("CacheSpec", ("batch", _i64), ("tokens", _i64), ("pages", _i64), ("max_pages", _i64), ("page", _i32), ("kv_heads", _i32), ("d", _i32), ("dtype", _i32),
                  *((n, Operand) for n in ("k", "v", "k_scale", "v_scale", "page_table", "lengths", "starts")))
CacheAppendSpec = _spec("CacheAppendSpec", ("cache", CacheSpec), ("dtype", _i32), ("heads", _i32), ("pairs", _i32), ("interleaved", _i32), ("magnitude", _f32),
                        ("frequencies", ctypes.POINTER(ctypes.c_double)), *((n, Operand) for n in ("positions", "k", "v", "q", "q_out")))
CacheAttentionSpec = _spec("CacheAttentionSpec", ("cache", CacheSpec), ("dtype", _i32), ("heads", _i32), ("scale", _f32), ("cap", _f32), ("window", _i64), ("sinks", _i64),
                           *((n, Operand) for n in ("q", "out", "lse", "slopes")))
SampleSpec = _spec("SampleSpec", ("rows", _i64), ("vocab", _i64), ("dtype", _i32), ("top_k", _i32), ("temperature", _f32), ("top_p", _f32), ("min_p", _f32),
                   *((n, Operand) for n in ("logits", "uniform", "temperatures", "top_ps", "min_ps", "top_ks", "tokens", "logprob")))
DTYPE = {"single": 0, "bfloat16": 1, "half": 2}   # B200_F32, B200_BF16, B200_F16
E4M3 = 3                                          # B200_E4M3: nodes of precision byte
MASKS = {"none": 0, "causal": 1, "prefix": 2}


class Operator:
    """A linked operator (`b200_operator`): `run` queues it on the device's stream.  Like a routine it keeps the addresses of
    its nodes; free it before their pools."""

    def __init__(self, device: Device, entry: str, spec):
        self.h = ctypes.c_void_p()
        check(getattr(lib(), entry)(device.h, ctypes.byref(spec), ctypes.byref(self.h)))
        self._run = lib().b200_operator_run

    def run(self):
        rc = self._run(self.h)
        if rc:
            check(rc)

    def free(self):
        if self.h:
            check(lib().b200_operator_free(self.h))
            self.h = None


def compile(ir: IrRoutine, options: Optional[str] = None) -> Code:  # noqa: A001 (mirrors Backend.compile)
    return Code(ir, options)


def rotary_frequencies(dims: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0, original: int = 4096,
                       fast: float = 32.0, slow: float = 1.0) -> Tuple[np.ndarray, float]:
    """Radians per position of the dims / 2 pairs of `Context.rotary`, and the magnitude: theta^(-2i / dims), for long contexts
    "linear" (positions shrink by `factor`), "ntk" (the base grows, so that the slowest pair shrinks by `factor` and the
    fastest stays) or "yarn" (pairs that turn more than `fast` times over the `original` context stay, those that turn less
    than `slow` times shrink by `factor`, a ramp between; magnitude 0.1 ln(factor) + 1)."""
    if dims < 0 or dims % 2 or theta <= 0 or factor <= 0:
        raise UserError(-5, "rotary_frequencies: an even number of dims, a positive base and factor")
    m = dims // 2
    i = np.arange(m, dtype=np.float64)
    f = theta ** (-i / max(m, 1))
    if scaling == "none":
        return f, 1.0
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "ntk":
        return (theta * factor ** (m / max(1, m - 1))) ** (-i / max(m, 1)), 1.0
    if scaling != "yarn":
        raise UserError(-5, "rotary_frequencies: unknown scaling '%s'" % scaling)
    low, high = (m * np.log(original / (2.0 * np.pi * turns)) / np.log(theta) for turns in (fast, slow))
    low, high = max(0.0, np.floor(low)), min(m - 1.0, np.ceil(high))
    ramp = np.clip((i - low) / max(1e-3, high - low), 0.0, 1.0)
    return f * (1.0 - ramp) + f / factor * ramp, float(0.1 * np.log(factor) + 1.0)


POOL_CAP = 0x1_0000_0000   # bytes per pool while offsets are 32-bit (arrayjit/lib/backends.ml:536)


def plan_pool_segments(items: Sequence[Tuple[int, int]], cap: int = POOL_CAP, what: str = "allocate_delta",
                       names: Optional[Sequence[str]] = None) -> Tuple[List[Tuple[int, int]], List[int]]:
    """`Backend_utils.plan_pool_segments` (arrayjit/lib/backends.ml:22-51): lays `(size, alignment)`
    items out in order; an item that would carry a pool past `cap` bytes opens a new pool at
    offset 0.  Returns `[(segment, offset)]` per item and the byte size of every segment; an item
    larger than the cap is a user error."""
    seg, bump, closed, out = 0, 0, [], []
    for i, (size, align) in enumerate(items):
        if size > cap:
            raise UserError(-5, "%s: tensor node %s needs %d bytes, over the %d-byte per-pool cap; set large_models" % (
                what, names[i] if names else i, size, cap))
        off = bump if align <= 1 else (bump + align - 1) // align * align
        if off + size > cap:
            closed.append(bump)
            seg += 1
            bump = size
            out.append((seg, 0))
        else:
            bump = off + size
            out.append((seg, off))
    return out, (closed + [bump]) if items else []


class Context:
    """`Backend_intf.context`: a device plus the {node -> (pool, offset)} map of the nodes it
    holds.  Contexts are persistent: `link` returns a routine whose `.context` is the child.

    `packing` chooses how `link` lays out the nodes the parent does not hold yet:
      "reference"  as `Raise_backend.allocate_delta` does (arrayjit/lib/backends.ml:529-614): working
                   nodes and read-only nodes go to separate pools, every node aligned to its ELEMENT
                   size only, pools cut at 4 GiB unless `large_models`, read-only nodes shared per
                   device by identifier;
      "aligned"    one pool, every node at a multiple of 256 bytes (the default of this mirror:
                   every stage then keeps its fastest form)."""

    def __init__(self, device: Device, arrays: Optional[Dict[str, Tuple[int, int, Tnode]]] = None,
                 packing: str = "aligned", large_models: bool = False):
        self.device = device
        self.arrays: Dict[str, Tuple[int, int, Tnode]] = dict(arrays or {})   # ident -> (pool, offset, tn)
        self.packing = packing
        self.large_models = large_models

    def _child(self, arrays) -> "Context":
        return Context(self.device, arrays, self.packing, self.large_models)

    def allocate(self, tnodes: Sequence[Tnode]) -> "Context":
        """Child context that also holds `tnodes`, packed back to back in one new zeroed pool
        (how the data-parallel driver keeps all gradients in one contiguous range)."""
        new = [t for t in tnodes if t.ident not in self.arrays]
        arrays = dict(self.arrays)
        if new:
            offs, total = [], 0
            for t in new:
                total = (total + 255) // 256 * 256
                offs.append(total)
                total += t.size_in_bytes
            pool = self.device.alloc_pool(max(total, 1))
            self.device.memset_zero(pool, 0, max(total, 1))
            for t, o in zip(new, offs):
                arrays[t.ident] = (pool, o, t)
        return self._child(arrays)

    def _pack_reference(self, group: List[Tnode], arrays, zero: bool = True):
        if not group:
            return
        cap = (1 << 62) if self.large_models else POOL_CAP
        items = [(t.size_in_bytes, PREC_BYTES[t.prec]) for t in group]
        where, sizes = plan_pool_segments(items, cap, "allocate_delta", [t.ident for t in group])
        pools = []
        for seg, size in enumerate(sizes):
            align = max(PREC_BYTES[t.prec] for t, (s, _) in zip(group, where) if s == seg)
            pools.append(self.device.alloc_pool(max(size, 1), alignment=align))
        for t, (seg, off) in zip(group, where):
            if zero and not t.zero_init:
                self.device.memset_zero(pools[seg], off, t.size_in_bytes)
            arrays[t.ident] = (pools[seg], off, t)

    def link(self, code: Code) -> "Routine":
        dev = self.device
        new: List[Tnode] = [t for t in code.ir.params() if t.ident not in self.arrays]
        arrays = dict(self.arrays)
        if new and self.packing == "reference":
            cache = dev.__dict__.setdefault("constant_buffer_cache", {})
            working = [t for t in new if not t.read_only]
            constants = [t for t in new if t.read_only]
            self._pack_reference(working, arrays)
            fresh = []
            for t in constants:
                hit = cache.get(t.ident)
                if hit is not None and hit[2].prec == t.prec and tuple(hit[2].dims) == tuple(t.dims):
                    arrays[t.ident] = hit
                else:
                    fresh.append(t)
            self._pack_reference(fresh, arrays)
            for t in fresh:
                cache[t.ident] = arrays[t.ident]
        elif new:
            # bump-pack the delta into one pool at 256-byte multiples
            offs, total = [], 0
            for t in new:
                align = 256
                total = (total + align - 1) // align * align
                offs.append(total)
                total += t.size_in_bytes
            pool = dev.alloc_pool(max(total, 1))
            dev.memset_zero(pool, 0, max(total, 1))
            for t, o in zip(new, offs):
                arrays[t.ident] = (pool, o, t)
        for t in code.ir.params():
            have = arrays[t.ident][2]
            if have.prec != t.prec or tuple(have.dims) != tuple(t.dims):
                raise UserError(-5, "link: node '%s' is held with another precision or shape" % t.ident)
        params = code.ir.params()
        binds = (Binding * max(len(params), 1))()
        for i, t in enumerate(params):
            pool, off, _ = arrays[t.ident]
            binds[i] = Binding(t.id, pool, off)
        h = ctypes.c_void_p()
        check(lib().b200_link(dev.h, code.h, binds, ctypes.c_int(len(params)), ctypes.byref(h)))
        return Routine(self._child(arrays), code, h)

    # ---- operators over nodes of this context (b200_layer_norm_link and its kin in include/b200.h, which define them)
    def _operand(self, what: str, ident: Optional[str], prec, dims) -> Operand:
        """The node's location, its precision and shape checked; dims None: any, "*" in dims: any extent."""
        if ident is None:
            return Operand(-1, 0)
        if ident not in self.arrays:
            raise UserError(-5, "%s: the context holds no node '%s'" % (what, ident))
        pool, off, t = self.arrays[ident]
        if t.prec not in ((prec,) if isinstance(prec, str) else prec):
            raise UserError(-5, "%s: node '%s' is of precision %s, not %s" % (what, ident, t.prec, prec))
        if dims is not None and tuple(t.dims) != tuple(dims):
            raise UserError(-5, "%s: node '%s' has dims %s, not %s" % (what, ident, tuple(t.dims), tuple(dims)))
        return Operand(pool, off)

    def _node(self, what: str, ident: str) -> Tnode:
        if ident not in self.arrays:
            raise UserError(-5, "%s: the context holds no node '%s'" % (what, ident))
        t = self.arrays[ident][2]
        if t.prec not in DTYPE:
            raise UserError(-5, "%s: node '%s' of precision %s: single, bfloat16 or half is wanted" % (what, ident, t.prec))
        return t

    def _norm(self, what: str, x: str, gamma: Optional[str], beta: Optional[str], eps: float, rows_like, weights, stats, sums) -> Operator:
        t = self._node(what, x)
        if not t.dims:
            raise UserError(-5, "%s: node '%s' has no axis" % (what, x))
        n = t.dims[-1]
        given = {self._node(what, w).prec for w in (gamma, beta) if w is not None}
        if len(given) > 1:
            raise UserError(-5, "%s: gamma and beta are of one precision" % what)
        wprec = given.pop() if given else "single"
        spec = LayerNormSpec(rows=t.num_elems // n if n else 0, n=n, dtype=DTYPE[t.prec], weight_dtype=DTYPE[wprec], eps=eps)
        for names, prec, dims in ((dict(rows_like, x=x), t.prec, t.dims), (weights, wprec, (n,)), (stats, "single", t.dims[:-1]),
                                  (sums, "single", (n,))):
            for field, ident in names.items():
                setattr(spec, field, self._operand(what, ident, prec, dims))
        return Operator(self.device, "b200_%s_link" % what, spec)

    def layer_norm(self, x: str, y: str, gamma: Optional[str] = None, beta: Optional[str] = None, residual: Optional[str] = None,
                   total: Optional[str] = None, mean: Optional[str] = None, rstd: Optional[str] = None, eps: float = 1e-5) -> Operator:
        """y = the norm of x (+ residual, their sum kept in `total`) along the last axis, scaled by gamma, shifted by beta.
        mean, rstd (single, the shape of x without its last axis) are what `layer_norm_grad` reads."""
        return self._norm("layer_norm", x, gamma, beta, eps, dict(y=y, residual=residual, total=total), dict(gamma=gamma, beta=beta),
                          dict(mean=mean, rstd=rstd), {})

    def layer_norm_grad(self, x: str, dy: str, dx: str, mean: str, rstd: str, gamma: Optional[str] = None, dgamma: Optional[str] = None,
                        dbeta: Optional[str] = None, d_total: Optional[str] = None) -> Operator:
        """The gradients of `layer_norm`: x is its input, `total` where there was a residual (whose gradient is dx too);
        d_total is added to dx; dgamma and dbeta (single) are sums over all rows."""
        return self._norm("layer_norm_grad", x, gamma, None, 0.0, dict(dy=dy, dx=dx, d_total=d_total), dict(gamma=gamma),
                          dict(mean=mean, rstd=rstd), dict(dgamma=dgamma, dbeta=dbeta))

    def rotary(self, tensors: Sequence[Tuple[str, str]], frequencies: Sequence[float], magnitude: float = 1.0,
               positions: Optional[str] = None, first_position: int = 0, layout: str = "half", inverse: bool = False) -> Operator:
        """Turns the pairs of one or two tensors [batch, seq, heads, d], given as (from, to) (which may be one node), by
        position * frequencies[pair] (radians, `rotary_frequencies`).  layout: "half" pairs element i with
        i + len(frequencies), "interleaved" 2i with 2i + 1.  inverse: the other way, as gradients go."""
        if not 1 <= len(tensors) <= 2:
            raise UserError(-5, "rotary: one or two tensors")
        if layout not in ("half", "interleaved"):
            raise UserError(-5, "rotary: unknown layout '%s'" % layout)
        t = self._node("rotary", tensors[0][0])
        if len(t.dims) != 4:
            raise UserError(-5, "rotary: node '%s' is not [batch, seq, heads, d]" % tensors[0][0])
        f = np.ascontiguousarray(frequencies, dtype=np.float64).reshape(-1)
        spec = RotarySpec(batch=t.dims[0], seq=t.dims[1], d=t.dims[3], pairs=f.size, dtype=DTYPE[t.prec], interleaved=int(layout == "interleaved"),
                          inverse=int(inverse), magnitude=magnitude, frequencies=f.ctypes.data_as(ctypes.POINTER(ctypes.c_double)),
                          first_position=first_position, positions=self._operand("rotary", positions, "int32", t.dims[:2]))
        for i, (src, dst) in enumerate(tensors):
            u = self._node("rotary", src)
            dims = (t.dims[0], t.dims[1], u.dims[2] if len(u.dims) == 4 else -1, t.dims[3])
            spec.heads[i] = dims[2]
            spec.x[i], spec.y[i] = self._operand("rotary", src, t.prec, dims), self._operand("rotary", dst, t.prec, dims)
        return Operator(self.device, "b200_rotary_link", spec)

    def _attention(self, what: str, q: str, k: str, rows_like, keys_like, lse, mask, prefix, documents, lengths, slopes, scale, cap) -> Operator:
        t, u = self._node(what, q), self._node(what, k)
        if len(t.dims) != 4 or len(u.dims) != 4:
            raise UserError(-5, "%s: q is [batch, queries, heads, d], k and v are [batch, keys, kv_heads, d]" % what)
        if mask not in MASKS:
            raise UserError(-5, "%s: unknown mask '%s'" % (what, mask))
        (b, s, h, d), (n, hk) = t.dims, u.dims[1:3]
        spec = AttentionSpec(batch=b, queries=s, keys=n, heads=h, kv_heads=hk, d=d, dtype=DTYPE[t.prec], mask=MASKS[mask],
                             scale=1.0 / np.sqrt(d) if scale is None and d else scale or 0.0, cap=cap)
        qdoc, kdoc = (None, documents) if documents is None or isinstance(documents, str) else documents
        for names, prec, dims in ((dict(rows_like, q=q), t.prec, t.dims), (dict(keys_like, k=k), t.prec, (b, n, hk, d)),
                                  (dict(lse=lse), "single", (b, h, s)), (dict(prefix=prefix, lengths=lengths), "int32", (b,)),
                                  (dict(query_documents=qdoc), "int32", (b, s)), (dict(key_documents=kdoc), "int32", (b, n)),
                                  (dict(slopes=slopes), "single", (h,))):
            for field, ident in names.items():
                setattr(spec, field, self._operand(what, ident, prec, dims))
        return Operator(self.device, "b200_%s_link" % what, spec)

    def attention(self, q: str, k: str, v: str, out: str, lse: Optional[str] = None, mask: str = "causal", prefix: Optional[str] = None,
                  documents=None, lengths: Optional[str] = None, slopes: Optional[str] = None, scale: Optional[float] = None,
                  cap: float = 0.0) -> Operator:
        """out = softmax over the visible keys of the scores, times v; lse (single [batch, heads, queries]) is what
        `attention_grad` reads.  The queries are the last ones of each sequence's `lengths` (or all) keys.  mask: "none",
        "causal" or "prefix" (keys before prefix[b] are seen by all).  documents: an int32 node of numbers per key, where
        a query has the number of the key at its position -- or two nodes, of queries and keys; queries see keys of their own document, a
        negative number is padding.  slopes: bias by distance,
        -slopes[h] * |position - key|.  scale: 1 / sqrt(d) by default.  cap: scores become cap * tanh(score / cap)."""
        return self._attention("attention", q, k, dict(out=out), dict(v=v), lse, mask, prefix, documents, lengths, slopes, scale, cap)

    def attention_grad(self, q: str, k: str, v: str, out: str, lse: str, d_out: str, dq: str, dk: str, dv: str, mask: str = "causal",
                       prefix: Optional[str] = None, documents=None, lengths: Optional[str] = None, slopes: Optional[str] = None,
                       scale: Optional[float] = None, cap: float = 0.0) -> Operator:
        """The gradients of `attention`, from its inputs, its out and lse, and the gradient d_out of out."""
        return self._attention("attention_grad", q, k, dict(out=out, d_out=d_out, dq=dq), dict(v=v, dk=dk, dv=dv), lse, mask, prefix,
                               documents, lengths, slopes, scale, cap)

    def _cache(self, what: str, prec: str, d: int, tokens: int, k_cache: str, v_cache: str, pages: str, lengths: str, starts, k_scale, v_scale) -> CacheSpec:
        for n in (k_cache, pages, lengths):
            if n not in self.arrays:
                raise UserError(-5, "%s: the context holds no node '%s'" % (what, n))
        c, table = self.arrays[k_cache][2], self.arrays[pages][2]
        if len(c.dims) != 4 or c.dims[3] != d:
            raise UserError(-5, "%s: node '%s' is not [pages, kv_heads, page, %d]" % (what, k_cache, d))
        if len(table.dims) != 2:
            raise UserError(-5, "%s: node '%s' is not [batch, max_pages]" % (what, pages))
        coded = k_scale is not None or v_scale is not None
        if coded and (k_scale is None or v_scale is None):
            raise UserError(-5, "%s: k_scale and v_scale go together" % what)
        (n, hk, page, _), b = c.dims, table.dims[0]
        spec = CacheSpec(batch=b, tokens=tokens, pages=n, max_pages=table.dims[1], page=page, kv_heads=hk, d=d, dtype=E4M3 if coded else DTYPE[prec])
        for names, p, dims in ((dict(k=k_cache, v=v_cache), "byte" if coded else prec, c.dims), (dict(k_scale=k_scale, v_scale=v_scale), "single", (n, hk)),
                               (dict(page_table=pages), "int32", table.dims), (dict(lengths=lengths), "int32", (b,)), (dict(starts=starts), "int32", (b + 1,))):
            for field, ident in names.items():
                setattr(spec, field, self._operand(what, ident, p, dims))
        return spec

    def _rows_of_heads(self, what: str, ident: str) -> Tnode:
        t = self._node(what, ident)
        if len(t.dims) != 3:
            raise UserError(-5, "%s: node '%s' is not [tokens, heads, d]" % (what, ident))
        return t

    def cache_append(self, k: str, v: str, k_cache: str, v_cache: str, pages: str, lengths: str, starts: Optional[str] = None,
                     k_scale: Optional[str] = None, v_scale: Optional[str] = None, q: Optional[str] = None, q_out: Optional[str] = None,
                     frequencies: Sequence[float] = (), magnitude: float = 1.0, positions: Optional[str] = None, layout: str = "half") -> Operator:
        """New keys and values [tokens, kv_heads, d] go to their slots of a cache in pages [pages, kv_heads, page, d]; the keys, and queries
        q [tokens, heads, d] (to q_out, which may be q), turn by their positions on the way as in `rotary` (no frequencies: they do not).
        pages: an int32 node [batch, max_pages] of page numbers, lengths: int32 [batch], the new tokens included; starts: int32 [batch + 1],
        the first row of each sequence's new tokens (without: as many rows each).  positions: int32 [tokens], others to turn by.
        k_scale, v_scale: single nodes [pages, kv_heads]; with them the caches are nodes of precision byte that hold e4m3 codes."""
        what = "cache_append"
        if layout not in ("half", "interleaved"):
            raise UserError(-5, "%s: unknown layout '%s'" % (what, layout))
        if (q is None) != (q_out is None):
            raise UserError(-5, "%s: q and q_out go together" % what)
        t = self._rows_of_heads(what, k)
        n, hk, d = t.dims
        f = np.ascontiguousarray(frequencies, dtype=np.float64).reshape(-1)
        spec = CacheAppendSpec(dtype=DTYPE[t.prec], pairs=f.size, interleaved=int(layout == "interleaved"), magnitude=magnitude,
                               frequencies=f.ctypes.data_as(ctypes.POINTER(ctypes.c_double)), positions=self._operand(what, positions, "int32", (n,)),
                               k=self._operand(what, k, t.prec, (n, hk, d)), v=self._operand(what, v, t.prec, (n, hk, d)))
        if q is not None:
            dims = (n, self._rows_of_heads(what, q).dims[1], d)
            spec.heads, spec.q, spec.q_out = dims[1], self._operand(what, q, t.prec, dims), self._operand(what, q_out, t.prec, dims)
        spec.cache = self._cache(what, t.prec, d, n, k_cache, v_cache, pages, lengths, starts, k_scale, v_scale)
        if spec.cache.kv_heads != hk:
            raise UserError(-5, "%s: node '%s' has %d heads, the cache %d" % (what, k, hk, spec.cache.kv_heads))
        return Operator(self.device, "b200_cache_append_link", spec)

    def cache_attention(self, q: str, k_cache: str, v_cache: str, out: str, pages: str, lengths: str, starts: Optional[str] = None,
                        k_scale: Optional[str] = None, v_scale: Optional[str] = None, lse: Optional[str] = None, window: int = 0, sinks: int = 0,
                        slopes: Optional[str] = None, scale: Optional[float] = None, cap: float = 0.0) -> Operator:
        """Attention of new tokens q [tokens, heads, d] over a cache in pages that holds them (`cache_append`, which describes the cache's nodes).
        A token sees those at its position and before it: all, or, with a window, the last `window` of them and the first `sinks`.
        lse: single [tokens, heads].  slopes, scale, cap: as in `attention`."""
        what = "cache_attention"
        t = self._rows_of_heads(what, q)
        n, h, d = t.dims
        spec = CacheAttentionSpec(dtype=DTYPE[t.prec], heads=h, scale=1.0 / np.sqrt(d) if scale is None and d else scale or 0.0, cap=cap, window=window, sinks=sinks,
                                  q=self._operand(what, q, t.prec, t.dims), out=self._operand(what, out, t.prec, t.dims),
                                  lse=self._operand(what, lse, "single", (n, h)), slopes=self._operand(what, slopes, "single", (h,)),
                                  cache=self._cache(what, t.prec, d, n, k_cache, v_cache, pages, lengths, starts, k_scale, v_scale))
        return Operator(self.device, "b200_cache_attention_link", spec)

    def sample(self, logits: str, uniform: str, tokens: str, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, logprob: Optional[str] = None) -> Operator:
        """Chooses a token (int32 node `tokens`) for each row of logits [.., vocab] by the random number in [0, 1) of the single node
        `uniform`, among the top_k largest (0: all) of them, the fewest that have top_p of their sum, and those of at least min_p times
        the largest probability.  temperature 0: the largest.  Each setting is a number or a node of one a row (single, top_k int32).
        logprob (single): the logarithm of the probability that the token had among those kept."""
        what = "sample"
        t = self._node(what, logits)
        if not t.dims:
            raise UserError(-5, "%s: node '%s' has no axis" % (what, logits))
        rows, vocab = t.dims[:-1], t.dims[-1]
        spec = SampleSpec(rows=t.num_elems // vocab if vocab else 0, vocab=vocab, dtype=DTYPE[t.prec], temperature=1.0, top_p=1.0,
                          logits=self._operand(what, logits, t.prec, t.dims), uniform=self._operand(what, uniform, "single", rows),
                          tokens=self._operand(what, tokens, "int32", rows), logprob=self._operand(what, logprob, "single", rows))
        for field, value, prec in (("temperature", temperature, "single"), ("top_k", top_k, "int32"), ("top_p", top_p, "single"), ("min_p", min_p, "single")):
            if isinstance(value, str):
                setattr(spec, field + "s", self._operand(what, value, prec, rows))
            else:
                setattr(spec, field, max(-1, min(value, 2 ** 31 - 1)) if field == "top_k" else value)
        return Operator(self.device, "b200_sample_link", spec)

    # ---- host access (Context.set_values / get_values, arrayjit/lib/context.ml:322-395)
    def from_host(self, ident: str, arr: np.ndarray):
        pool, off, t = self.arrays[ident]
        words = 4 if t.prec == "uint4x32" else 1
        a = np.ascontiguousarray(arr, dtype=np.uint32 if words == 4 else NP_DTYPE[t.prec]).reshape(-1)
        if a.size != t.num_elems * words:
            raise UserError(-5, "from_host: '%s' has %d elements, got %d" % (ident, t.num_elems, a.size))
        self.device.from_host(pool, off, a)
        self.device.await_()     # the staging array may be a temporary

    def to_host(self, ident: str) -> np.ndarray:
        pool, off, t = self.arrays[ident]
        out = np.empty(t.dims if t.dims else (1,), NP_DTYPE[t.prec])
        self.device.to_host(pool, off, out)
        self.device.await_()
        return out


class Routine:
    """`Backend_intf.routine`: a linked routine; `run` schedules it on the device stream
    (`Task.run routine.schedule`, lib/train.ml:42)."""

    def __init__(self, context: Context, code: Code, h):
        self.context = context
        self.code = code
        self.h = h
        self.static_syms = [s for s, _ in code.ir.static]

    def run(self, **static):
        n = len(self.static_syms)
        vals = (ctypes.c_int64 * max(n, 1))(*[int(static[s]) for s in self.static_syms])
        check(lib().b200_launch(self.h, vals, ctypes.c_int(n)))

    def info(self) -> dict:
        """The plan that runs: the code's, or a re-planned variant of it when the bound addresses
        ruled out a stage's aligned form (b200_routine_info)."""
        buf = ctypes.create_string_buffer(1 << 16)
        check(lib().b200_routine_info(self.h, buf, ctypes.c_size_t(1 << 16)))
        return json.loads(buf.value.decode())

    def use_graph(self, on: bool = True):
        check(lib().b200_routine_use_graph(self.h, ctypes.c_int(int(on))))

    def kernels_per_run(self) -> int:
        k = ctypes.c_int64(0)
        check(lib().b200_routine_launch_count(self.h, ctypes.byref(k)))
        return k.value

    def profile(self, on: bool = True):
        check(lib().b200_routine_profile(self.h, ctypes.c_int(int(on))))

    def stage_times(self):
        """[(total_ms, runs)] per stage, over the runs made while profiling was on; 0 runs for a stage in the launch
        of another, whose time includes it."""
        out = []
        for i in range(len(self.info()["stages"])):
            ms, n = ctypes.c_float(0), ctypes.c_int(0)
            check(lib().b200_routine_stage_time(self.h, ctypes.c_int(i), ctypes.byref(ms), ctypes.byref(n)))
            out.append((ms.value, n.value))
        return out

    def free(self):
        if self.h:
            lib().b200_routine_free(self.h)
            self.h = None
