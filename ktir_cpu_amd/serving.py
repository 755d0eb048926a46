"""Operators of a served model's layer on device arrays: rotary positions, a
key / value cache in 8 bits, and attention over it.

They stand next to the launches that KTIR functions become, for programs that
keep their tensors on the device: each class checks its arrays once, builds the
descriptor of its entry point in ``include/ktir_hip.h`` and launches it with
``run()``, as often as the program likes, on whatever the arrays then hold.

    cache = KV8Cache(k_codes, v_codes, k_scale, v_scale)
    turn = Rope(q, positions, freq, q_rot, k=k, k_out=k_rot)
    keep = KV8Append(cache, k_rot, v, table, q_start, kv_len)
    attend = KV8Attention(cache, q_rot, out, table, q_start, kv_len, max_q=1, max_k=8192)
    for each step: ...; turn.run(); keep.run(); attend.run()

Arrays are torch tensors on the library's device, :class:`DeviceArray`, or any
object with ``__cuda_array_interface__`` (bf16 as uint16, e4m3 codes as uint8, as
arrays travel elsewhere in this package).  The last dimension is contiguous;
other strides are free within the limits that the header names.

Streams: ``run(stream)`` launches on a torch stream of the library's device or a raw
handle (0 is the null stream).  Without one, a launch on torch tensors goes to torch's current
stream, so it is ordered with the torch operations around it and can be captured
into a graph; a launch on other arrays goes to the library's stream, as all else
here.  Nothing waits: ``runtime.sync()`` waits for the library's stream, and
reports lengths and tables that were out of range (IndexError) whatever stream
found them, once that stream is done.  One handle is run by one thread at a time,
and its runs do not overlap on the device; it and its arrays live until the last of
them, or the last replay of a graph that holds one, is done.
"""

from __future__ import annotations

import ctypes as C
import sys
from typing import NamedTuple, Optional, Tuple

import numpy as np

from . import runtime as rt

_TORCH = {"torch.float16": "f16", "torch.bfloat16": "bf16", "torch.float32": "f32", "torch.float64": "f64",
          "torch.int8": "i8", "torch.float8_e4m3fn": "e4m3", "torch.int32": "i32", "torch.int64": "i64",
          "torch.uint8": "u8"}
_TYPESTR = {"<f2": "f16", "<u2": "bf16", "<f4": "f32", "<f8": "f64", "|i1": "i8", "|u1": "e4m3", "<i4": "i32",
            "<i8": "i64"}


_NULL_STREAM = rt.K["KTIR_STREAM_NULL"]


class DeviceArray:
    """A C-contiguous array in device memory of the library, from a host array."""

    def __init__(self, host: np.ndarray):
        host = np.ascontiguousarray(host)
        self.shape, self.dtype = host.shape, host.dtype
        self.buffer = rt.DeviceBuffer(host.nbytes)
        self.put(host)

    @property
    def __cuda_array_interface__(self):
        return dict(shape=self.shape, typestr=self.dtype.str, version=2, strides=None, data=(self.buffer.ptr, False))

    def put(self, host: np.ndarray):
        """Overwrite the array (waits for the library's stream)."""
        host = np.ascontiguousarray(host, dtype=self.dtype)
        if host.shape != self.shape:
            raise ValueError(f"an array of shape {host.shape} into one of {self.shape}")
        self.buffer.upload(host)

    def numpy(self) -> np.ndarray:
        """The array's values, after what the library's stream holds."""
        out = np.empty(self.shape, self.dtype)
        self.buffer.download_into(out)
        return out


class _View(NamedTuple):
    ptr: int
    dtype: str
    shape: Tuple[int, ...]
    strides: Tuple[int, ...]        # in elements
    device: Optional[int]           # torch's device index; None: not a torch tensor


def _view(x, name: str, ndim: int, dtypes, dense: bool = True) -> _View:
    """Where an array lies, checked for its rank and type and (dense) a contiguous last dimension."""
    if hasattr(x, "data_ptr") and hasattr(x, "stride"):
        if x.device.type != "cuda":
            raise ValueError(f"{name}: a tensor on {x.device}; it has to be on the GPU")
        dtype = _TORCH.get(str(x.dtype))
        v = _View(x.data_ptr(), dtype or str(x.dtype), tuple(x.shape), tuple(x.stride()), x.device.index or 0)
    else:
        try:
            a = x.__cuda_array_interface__
        except AttributeError:
            raise TypeError(f"{name}: {type(x).__name__} is no device array (a torch tensor, a DeviceArray, or one "
                            "with __cuda_array_interface__)") from None
        typestr, shape = a["typestr"], tuple(int(n) for n in a["shape"])
        size = int(typestr[2:])
        if a.get("strides") is None:
            strides = [1] * len(shape)
            for i in range(len(shape) - 2, -1, -1):
                strides[i] = strides[i + 1] * shape[i + 1]
        else:
            if any(s % size for s in a["strides"]):
                raise ValueError(f"{name}: strides {a['strides']} are no multiples of {size} bytes")
            strides = [s // size for s in a["strides"]]
        v = _View(int(a["data"][0]), _TYPESTR.get(typestr, typestr), shape, tuple(strides), None)
    if len(v.shape) != ndim:
        raise ValueError(f"{name}: shape {v.shape}, not of {ndim} dimensions")
    if v.dtype not in dtypes:
        raise ValueError(f"{name}: type {v.dtype}, not {' or '.join(dtypes)}")
    if dense and v.shape[-1] > 1 and v.strides[-1] != 1:
        raise ValueError(f"{name}: its last dimension has stride {v.strides[-1]}, not 1")
    if any(s < 0 for s in v.strides):
        raise ValueError(f"{name}: a negative stride ({v.strides})")
    return v


def _same(name: str, got, want):
    if tuple(got) != tuple(want):
        raise ValueError(f"{name}: shape {tuple(got)}, not {tuple(want)}")


def _rows3(v: _View) -> rt.Rows3:
    return rt.Rows3(v.ptr, v.strides[0], v.strides[1])


class _Launch:
    """A checked descriptor and the arrays it points into."""

    entry = ""

    def __init__(self, desc, views, keep):
        self.desc = desc
        self._keep = keep               # what the descriptor's addresses belong to
        self._ref = C.byref(desc)
        self._call = None
        self._own, self._streams = None, None       # own workspace; where it is a torch tensor, the streams that it was used on
        devices = {v.device for v in views if v.device is not None}
        if len(devices) > 1:
            raise ValueError(f"{self.entry}: tensors on devices {sorted(devices)}")
        self._torch_device = devices.pop() if devices else None

    def _first(self):
        lib = rt.lib()
        if self._torch_device is not None and self._torch_device != rt.device_index():
            raise ValueError(f"{self.entry}: tensors on device {self._torch_device}; the library runs on device "
                             f"{rt.device_index()} (KTIR_DEVICE)")
        if self._torch_device is not None:
            torch = sys.modules["torch"]
            # the handle alone: 0.1 us, where a Stream object takes 1.1 of the 5 that a launch costs the host
            self._current = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
                lambda device: torch.cuda.current_stream(device).cuda_stream)
        self._call = getattr(lib, self.entry)

    def run(self, stream=None):
        """Launch on `stream` (see the module's notes); returns without waiting."""
        if self._call is None:
            self._first()
        if stream is not None:
            self.desc.stream = int(getattr(stream, "cuda_stream", stream)) or _NULL_STREAM
        elif self._torch_device is not None:
            self.desc.stream = self._current(self._torch_device) or _NULL_STREAM
        else:
            self.desc.stream = 0
        rc = self._call(self._ref)
        if rc:
            rt.check(rc)
        if self._streams is not None and self.desc.stream not in self._streams:
            self._used_on(stream)

    def _used_on(self, stream):
        """The own workspace came from torch: it goes to no other tensor before this stream is done with it.
        A raw handle is not recorded (its stream may end before the workspace does): its caller waits."""
        if stream is not None and not hasattr(stream, "cuda_stream"):
            return
        torch = sys.modules["torch"]
        if torch.cuda.is_current_stream_capturing():
            return                                  # (a replay's stream is not known here)
        self._own.record_stream(torch.cuda.current_stream(self._torch_device) if stream is None else stream)
        self._streams.add(self.desc.stream)


# ---- rotary positions --------------------------------------------------------

def rope_frequencies(rot: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                     trained: int = 4096, fast: float = 32.0, slow: float = 1.0,
                     divisors=None) -> Tuple[np.ndarray, float]:
    """Radians per position of the rot / 2 pairs (float64), and the amplitude.

    f_i = base^(-2 i / rot), and for contexts `factor` times the `trained` length:
      linear      f_i / factor
      ntk         the base grows by factor^(rot / (rot - 2)): the slowest pair slows by factor
      yarn        pairs of more than `fast` turns in the trained length keep f_i, those of fewer than
                  `slow` get f_i / factor, with a ramp over the pair's number between; the amplitude
                  is 0.1 ln(factor) + 1
      wavelength  as yarn, but the ramp goes over the turns themselves and the amplitude stays 1
    `divisors` (one per pair) divide f_i after that.
    """
    if rot < 2 or rot % 2:
        raise ValueError(f"rope_frequencies: {rot} columns (an even number of them is rotated)")
    if not (base > 0 and factor > 0 and trained > 0 and fast > 0 and slow > 0):
        raise ValueError("rope_frequencies: base, factor, trained, fast and slow are positive")
    i = np.arange(rot // 2, dtype=np.float64)
    if scaling == "ntk" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = np.float64(base) ** (-2.0 * i / rot)
    amplitude = 1.0
    if scaling in ("yarn", "wavelength"):
        if fast <= slow:
            raise ValueError(f"rope_frequencies: fast {fast} is not more than slow {slow}")
        if scaling == "yarn":
            def pair_of(turns):
                return rot * np.log(trained / (turns * 2 * np.pi)) / (2 * np.log(base))
            lo, hi = max(np.floor(pair_of(fast)), 0.0), min(np.ceil(pair_of(slow)), rot - 1.0)
            slowed = np.clip((i - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
            amplitude = float(0.1 * np.log(factor) + 1.0) if factor > 1 else 1.0
        else:
            slowed = np.clip((fast - trained * f / (2 * np.pi)) / (fast - slow), 0.0, 1.0)
        f = f * (1.0 - slowed) + f / factor * slowed
    elif scaling == "linear":
        f = f / factor
    elif scaling not in (None, "ntk"):
        raise ValueError(f"rope_frequencies: scaling {scaling!r}, not linear, ntk, yarn or wavelength")
    if divisors is not None:
        d = np.asarray(divisors, dtype=np.float64)
        _same("rope_frequencies: divisors", d.shape, f.shape)
        f = f / d
    return f, amplitude


class Rope(_Launch):
    """Rotary positions of `x` [tokens, heads, columns], and of `k` in the same launch.

    `positions` [tokens] int32 or int64, tokens at negative ones are skipped;
    `freq` [rot / 2] float64, radians per position: the first rot columns turn, the
    others are copied.  `out` / `k_out` None: in place.  `inverse` turns by the opposite
    angles, `amplitude` as it is: how a gradient of the output becomes one of the input,
    and the way back where the amplitude is 1.
    """

    entry = "ktir_launch_rope"

    def __init__(self, x, positions, freq, out=None, *, k=None, k_out=None, interleaved: bool = False,
                 amplitude: float = 1.0, inverse: bool = False):
        if k is None and k_out is not None:
            raise ValueError("Rope: k_out without k")
        a = _view(x, "x", 3, ("f16", "bf16", "f32"))
        b = a if out is None else _view(out, "out", 3, (a.dtype,))
        p = _view(positions, "positions", 1, ("i32", "i64"))
        f = _view(freq, "freq", 1, ("f64",))
        _same("out", b.shape, a.shape)
        _same("positions", p.shape, a.shape[:1])
        d = rt.Rope(tokens=a.shape[0], heads=a.shape[1], columns=a.shape[2], rot=2 * f.shape[0], in_=_rows3(a),
                    out=_rows3(b), pos=p.ptr, freq=f.ptr, amplitude=float(amplitude),
                    pos_dtype=rt.SERVING_CODE[p.dtype], dtype=rt.SERVING_CODE[a.dtype], interleaved=int(bool(interleaved)),
                    inverse=int(bool(inverse)))
        views = [a, b, p, f]
        if k is not None:
            c = _view(k, "k", 3, (a.dtype,))
            e = c if k_out is None else _view(k_out, "k_out", 3, (a.dtype,))
            _same("k", (c.shape[0], c.shape[2]), (a.shape[0], a.shape[2]))
            _same("k_out", e.shape, c.shape)
            d.heads2, d.in2, d.out2 = c.shape[1], _rows3(c), _rows3(e)
            views += [c, e]
        if d.rot > d.columns:
            raise ValueError(f"freq: {d.rot} columns to rotate of {d.columns}")
        super().__init__(d, views, (x, positions, freq, out, k, k_out))


# ---- the cache -------------------------------------------------------------------

class KV8Cache:
    """A paged key / value cache in 8 bits.

    `k`, `v` [pages, page, heads, columns] int8 or float8 (e4m3) codes, `k_scale`,
    `v_scale` [pages, heads] float32, not negative: a code stands for code * scale.  The page
    is a power of two from 16 to 256 tokens, columns a multiple of 16 up to 256.
    Neither needs initial values: a page's scale counts once tokens are in it.
    """

    def __init__(self, k, v, k_scale, v_scale):
        a = _view(k, "k", 4, ("i8", "e4m3"))
        b = _view(v, "v", 4, (a.dtype,))
        s, t = _view(k_scale, "k_scale", 2, ("f32",), False), _view(v_scale, "v_scale", 2, ("f32",), False)
        _same("v", b.shape, a.shape)
        _same("k_scale", s.shape, (a.shape[0], a.shape[2]))
        _same("v_scale", t.shape, (a.shape[0], a.shape[2]))
        self.desc = rt.KV8(a.ptr, b.ptr, s.ptr, t.ptr, a.shape[0], a.shape[1], a.shape[2], a.shape[3], *a.strides[:3],
                           *b.strides[:3], *s.strides, *t.strides, rt.SERVING_CODE[a.dtype], 0)
        self.views = [a, b, s, t]
        self.arrays = (k, v, k_scale, v_scale)


def _batch(table, q_start, kv_len, tokens: int):
    """The batch's descriptor, its views, and the number of sequences."""
    t, q, n = _view(table, "table", 2, ("i32",)), _view(q_start, "q_start", 1, ("i32",)), _view(kv_len, "kv_len", 1, ("i32",))
    seqs = n.shape[0]
    _same("q_start", q.shape, (seqs + 1,))
    if t.shape[0] != seqs:
        raise ValueError(f"table: {t.shape[0]} rows for {seqs} sequences")
    return rt.KV8Batch(t.ptr, q.ptr, n.ptr, seqs, tokens, t.strides[0], t.shape[1]), [t, q, n]


class KV8Append(_Launch):
    """New keys and values `k`, `v` [tokens, heads, columns] of a batch into the cache.

    Sequence s brings the tokens q_start[s] .. q_start[s + 1], the last of its
    kv_len[s] (int32, all on the device, read when the launch runs); its token t
    lies in page table[s, t // page].  Tokens outside every sequence pad the batch.
    No page is written for two places of the batch's tables at once.
    """

    entry = "ktir_launch_kv8_append"

    def __init__(self, cache: KV8Cache, k, v, table, q_start, kv_len):
        a = _view(k, "k", 3, ("f16", "bf16"))
        b = _view(v, "v", 3, (a.dtype,))
        _same("k", a.shape[1:], (cache.desc.heads, cache.desc.columns))
        _same("v", b.shape, a.shape)
        batch, views = _batch(table, q_start, kv_len, a.shape[0])
        d = rt.KV8Append(cache.desc, batch, _rows3(a), _rows3(b), 0, rt.SERVING_CODE[a.dtype], 0)
        super().__init__(d, [a, b, *views, *cache.views], (cache, k, v, table, q_start, kv_len))


class KV8Attention(_Launch):
    """Attention of the batch's new tokens over the cache, the tokens themselves
    (appended before) among it.

    `q`, `out` [tokens, query heads, columns]; consecutive query heads share a KV
    head.  `max_q`, `max_k`: the most new and cached tokens that a sequence of the
    batch has, over all runs.  `scale`: of the scores (columns^-1/2 if None).
    `window` > 0: a token sees that many tokens up to itself, and pages that end before
    the window of a sequence's first new token need no table entry.  `causal` False:
    every new token sees all cached ones.  `lse` [tokens, query heads] float32:
    the rows' log-sum-exp.  `workspace`: a device array of at least
    `workspace_bytes` bytes to use instead of an own one, which launches that
    follow one another on one stream may share.
    """

    entry = "ktir_launch_kv8_attention"

    def __init__(self, cache: KV8Cache, q, out, table, q_start, kv_len, *, max_q: int, max_k: int,
                 scale: Optional[float] = None, causal: bool = True, window: int = 0, lse=None, workspace=None):
        a = _view(q, "q", 3, ("f16", "bf16"))
        b = _view(out, "out", 3, (a.dtype,))
        _same("out", b.shape, a.shape)
        if a.shape[2] != cache.desc.columns:
            raise ValueError(f"q: {a.shape[2]} columns, the cache has {cache.desc.columns}")
        batch, views = _batch(table, q_start, kv_len, a.shape[0])
        d = rt.KV8Attn(cache=cache.desc, batch=batch, q=_rows3(a), out=_rows3(b), q_heads=a.shape[1], max_q=int(max_q),
                       max_k=int(max_k), window=int(window), scale=a.shape[2] ** -0.5 if scale is None else float(scale),
                       dtype=rt.SERVING_CODE[a.dtype], causal=int(bool(causal)))
        views += [a, b, *cache.views]
        if lse is not None:
            c = _view(lse, "lse", 2, ("f32",), False)
            _same("lse", c.shape, a.shape[:2])
            d.lse, d.lse_tok, d.lse_head = c.ptr, *c.strides
            views.append(c)
        rt.check(rt.opened().ktir_kv8_attention_plan(C.byref(d)))
        self.workspace_bytes = int(d.ws_bytes)
        if workspace is not None:
            w = _view(workspace, "workspace", 1, ("u8", "e4m3", "i8", "f32"))
            size = w.shape[0] * (4 if w.dtype == "f32" else 1)
            if size < self.workspace_bytes or w.ptr % 16:
                raise ValueError(f"workspace: {size} bytes at {w.ptr:#x}; it takes {self.workspace_bytes} on a 16-byte bound")
            d.ws = w.ptr
            views.append(w)
        super().__init__(d, views, (cache, q, out, table, q_start, kv_len, lse, workspace))
        if self.workspace_bytes and workspace is None:
            if self._torch_device is not None:
                torch = sys.modules["torch"]
                self._own = torch.empty(self.workspace_bytes, dtype=torch.uint8, device=f"cuda:{self._torch_device}")
                d.ws = self._own.data_ptr()
                self._streams = {torch.cuda.current_stream(self._torch_device).cuda_stream or _NULL_STREAM}
            else:
                self._own = rt.DeviceBuffer(self.workspace_bytes)
                d.ws = self._own.ptr
