"""The 4-bit KV cache: the buffers, the calls that write them, the attention that
reads them and the eviction that bounds them (C ABI: the hrm_kv4_* entry points
and hrm_split_gqkv_rope_kv4 of include/hrm_ops.h, where the format is defined).

A decode loop with a bounded cache, one step:

    gate, q, _, _ = split_gqkv_rope_kv4(gqkv, heads, cache, position, theta, table, cache_offset=rows, keep_kv=False)
    o = kv4_attention(q, cache, rows, gate=gate, accumulate=True)     # [b, s, h, d], gated
    rows = kv4_evict(cache, rows + s, budget, protect_from)           # int32 [b], back to at most budget

Offsets and lengths are ints, or int32 CUDA tensors with one value per sequence
(read on the device, so that a captured step can be replayed as they advance).

With `stream` a call is queued there, and the tensors that it makes belong to that
stream, as torch's own do under `with torch.cuda.stream(stream)`: another stream that
uses them waits for it first and, before it drops them, calls record_stream.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass, field
from typing import Optional, Tuple, Union

import torch

from ._lib import HRM_OK, LIB, Kv4CacheStruct, check
from .ops import _made, _need

GROUP = 32  # elements per (scale, base) pair
HEAD_DIMS = (64, 128, 192, 256)

Offset = Union[int, torch.Tensor]

# The handle of a device's current stream, without the Stream object around it (a
# decode step makes one such call per layer and operator).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _launch(name: str, device: torch.device, tensors, stream: Optional[torch.cuda.Stream], *args) -> None:
    """ops._launch for calls of a few microseconds: the same checks (every tensor and
    an explicit stream on `device`, which is current during the call), on plain
    integers."""
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"{name}: tensors on {device} and {t.device}; every argument must be on one device")
    if stream is None:
        handle = _raw_stream(device.index)
    elif stream.device != device:
        raise ValueError(f"{name}: stream on {stream.device} but tensors on {device}")
    else:
        handle = stream.cuda_stream
    if _current_device() == device.index:
        status = getattr(LIB, name)(*args, handle)
    else:
        with torch.cuda.device(device):
            status = getattr(LIB, name)(*args, handle)
    if status != HRM_OK:
        check(name, status)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


@dataclass(frozen=True, eq=False)
class Kv4Cache:
    """The buffers of one 4-bit cache (one layer's KV slot).

    k_codes, v_codes   uint8 [batch, kv_heads, cache_len, head_dim / 2]
    k_scales, v_scales bf16 [batch, kv_heads, cache_len, head_dim / 32, 2]
    weights            fp32 [batch, kv_heads, cache_len], or None
    positions          int32 [batch, kv_heads, cache_len], or None

    The shapes are checked here, once; the calls then pass the buffers as they
    are.  A cache's tensors cannot be replaced (make another one) and must not be
    resized; write into them to reset them.
    """

    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor
    weights: Optional[torch.Tensor] = None
    positions: Optional[torch.Tensor] = None
    shape: Tuple[int, int, int, int] = field(init=False, repr=False)

    def __post_init__(self):
        _need(self.k_codes, "k_codes", (torch.uint8,))
        if self.k_codes.dim() != 4 or 2 * self.k_codes.shape[3] not in HEAD_DIMS:
            raise ValueError("k_codes must be [batch, kv_heads, cache_len, head_dim / 2], head_dim 64, 128, 192 or 256")
        b, h, n, half = self.k_codes.shape
        put = object.__setattr__  # (frozen: the struct below holds these tensors' addresses)
        put(self, "shape", (b, h, n, 2 * half))
        want = {"v_codes": ((b, h, n, half), torch.uint8), "k_scales": ((b, h, n, 2 * half // GROUP, 2), torch.bfloat16),
                "v_scales": ((b, h, n, 2 * half // GROUP, 2), torch.bfloat16), "weights": ((b, h, n), torch.float32),
                "positions": ((b, h, n), torch.int32)}
        for name, (shape, dtype) in want.items():
            t = getattr(self, name)
            if t is None and name in ("weights", "positions"):
                continue
            _need(t, name, (dtype,))
            if tuple(t.shape) != shape:
                raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
            if t.device != self.k_codes.device:
                raise ValueError(f"{name} is on {t.device}, k_codes on {self.k_codes.device}")
        ptr = [None if t is None else t.data_ptr()
               for t in (self.k_codes, self.k_scales, self.v_codes, self.v_scales, self.weights, self.positions)]
        put(self, "_struct", Kv4CacheStruct(*ptr, b, h, n, 2 * half))
        put(self, "_ref", ctypes.pointer(self._struct))
        put(self, "device", self.k_codes.device)
        put(self, "_workspaces", {})  # bytes by (heads, seq, accumulate)


def kv4_cache(batch: int, kv_heads: int, cache_len: int, head_dim: int, device=None, track: bool = False) -> Kv4Cache:
    """A zeroed cache; track=True adds the weights and positions that kv4_evict needs."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim {head_dim}: the 4-bit cache takes {HEAD_DIMS}")
    d = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)

    def z(*tail, dtype):
        return torch.zeros((batch, kv_heads, cache_len, *tail), dtype=dtype, device=d)

    return Kv4Cache(z(head_dim // 2, dtype=torch.uint8), z(head_dim // GROUP, 2, dtype=torch.bfloat16),
                    z(head_dim // 2, dtype=torch.uint8), z(head_dim // GROUP, 2, dtype=torch.bfloat16),
                    z(dtype=torch.float32) if track else None, z(dtype=torch.int32) if track else None)


def _offset(x: Offset, name: str, batch: int):
    """(host value, tensor or None) of an int or an int32 CUDA tensor [batch]."""
    if not isinstance(x, torch.Tensor):
        return int(x), None
    _need(x, name, (torch.int32,))
    if x.numel() != batch:
        raise ValueError(f"{name} must have one value per sequence ({batch}), got {x.numel()}")
    return 0, x


def kv4_update(cache: Kv4Cache, k: torch.Tensor, v: torch.Tensor, position_offset: Offset = 0,
               cache_offset: Offset = 0, *, stream=None) -> Kv4Cache:
    """Writes k, v [batch, kv_heads, seq, head_dim] bf16 as cache rows cache_offset + s.

    The rows' weights become 0 and their positions position_offset + s.  The
    4-bit kv_cache_update (src/lib.rs:706-747).
    """
    _need(k, "k"); _need(v, "v")
    b, h, _, d = cache.shape
    if k.dim() != 4 or k.shape != v.shape or (k.shape[0], k.shape[1], k.shape[3]) != (b, h, d):
        raise ValueError(f"k and v must both be [{b}, {h}, seq, {d}]")
    pos, pos_t = _offset(position_offset, "position_offset", b)
    off, off_t = _offset(cache_offset, "cache_offset", b)
    _launch("hrm_kv4_update", cache.device, (k, v, pos_t, off_t), stream, cache._ref, _ptr(k), _ptr(v), k.shape[2], pos,
            _ptr(pos_t), off, _ptr(off_t))
    return cache


def _split_results(gqkv: torch.Tensor, b: int, s: int, h: int, d: int, keep_kv: bool):
    gate, q = gqkv.new_empty((b, s, h, d)), gqkv.new_empty((b, h, s, d))
    return (gate, q, torch.empty_like(q), torch.empty_like(q)) if keep_kv else (gate, q, None, None)


def split_gqkv_rope_kv4(gqkv: torch.Tensor, num_heads: int, cache: Kv4Cache, position_offset: Offset = 0,
                        theta: float = 10000.0, table: Optional[torch.Tensor] = None, cache_offset: Offset = 0,
                        out=None, keep_kv: bool = True, *, stream=None):
    """split_gqkv_rope into a 4-bit cache: (gate [b, s, h, d], q, k, v [b, h, s, d]).

    gate and q are split_gqkv_rope's; k and v are the values that the cache now
    holds for these tokens (None with keep_kv=False).  `out`: the four buffers.
    """
    _need(gqkv, "gqkv")
    b, h, _, d = cache.shape
    if num_heads != h or gqkv.dim() != 3 or gqkv.shape[0] != b or gqkv.shape[2] != 4 * h * d:
        raise ValueError(f"gqkv must be [{b}, seq, 4 * {h} * {d}] for this cache (num_heads {h})")
    s = gqkv.shape[1]
    if out is None:
        gate, q, k, v = _made(stream, _split_results, gqkv, b, s, h, d, keep_kv)
        given = ()
    else:
        gate, q, k, v = given = tuple(out)
        for t, n in zip(given, ("gate", "q", "k", "v")):
            if t is None and n in ("k", "v"):
                continue
            _need(t, n)
            if t.numel() != b * s * h * d:
                raise ValueError(f"{n} has the wrong size")
    positions = 0
    if table is not None:
        _need(table, "table", (torch.float32,))
        if table.dim() != 2 or table.shape[1] != d:
            raise ValueError("table must be [positions, head_dim]")
        positions = table.shape[0]
    pos, pos_t = _offset(position_offset, "position_offset", b)
    off, off_t = _offset(cache_offset, "cache_offset", b)
    _launch("hrm_split_gqkv_rope_kv4", cache.device, (gqkv, table, pos_t, off_t, *given), stream, gqkv.data_ptr(),
            gate.data_ptr(), q.data_ptr(), _ptr(k), _ptr(v), cache._ref, s, pos, _ptr(pos_t), theta, _ptr(table),
            positions, off, _ptr(off_t))
    return gate, q, k, v


def kv4_attention(q: torch.Tensor, cache: Kv4Cache, cache_offset: Offset, *, gate: Optional[torch.Tensor] = None,
                  prefix_len: int = 0, scale: Optional[float] = None, accumulate: bool = False,
                  out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                  stream=None) -> torch.Tensor:
    """Attention of q [b, heads, s, d] over the cache; out [b, s, heads, d].

    cache_offset counts the rows before the queries' own tokens, which the cache
    already holds: query i sees rows j <= cache_offset + i, and those below
    prefix_len.  gate [b, s, heads, d] multiplies by its sigmoid; scale defaults
    to 1 / sqrt(head_dim); accumulate adds the probabilities to cache.weights.
    workspace: a uint8 tensor of at least kv4_attention_workspace bytes, else one is
    allocated for the call, on the launch's stream.  A sequence with a negative
    cache_offset whose queries see nothing gives 0.  A probability has 16 bits in the
    sum over v for up to 32 query rows of a kv head (heads / kv_heads * s), 8 above.
    src/lib.rs:632-704.
    """
    _need(q, "q")
    b, hk, _, d = cache.shape
    if q.dim() != 4 or q.shape[0] != b or q.shape[3] != d or q.shape[1] % hk or q.shape[1] == 0:
        raise ValueError(f"q must be [{b}, a multiple of {hk} heads, seq, {d}]")
    h, s = q.shape[1], q.shape[2]
    if gate is not None:
        _need(gate, "gate")
        if gate.numel() != q.numel():
            raise ValueError("gate has the wrong size")
    if out is None:
        out = _made(stream, q.new_empty, (b, s, h, d))
    else:
        _need(out, "out")
        if out.numel() != q.numel():
            raise ValueError("out has the wrong size")
    off, off_t = _offset(cache_offset, "cache_offset", b)
    if accumulate and cache.weights is None:
        raise ValueError("accumulate needs a cache with weights (kv4_cache(..., track=True))")
    nbytes = kv4_attention_workspace(cache, h, s, accumulate)
    if nbytes and workspace is None:
        workspace = _made(stream, torch.empty, nbytes, dtype=torch.uint8, device=q.device)
    elif workspace is not None:
        _need(workspace, "workspace", (torch.uint8,))
        nbytes = workspace.numel()
    _launch("hrm_kv4_attention", cache.device, (q, out, gate, off_t, workspace), stream, _ptr(q), cache._ref,
            _ptr(gate), _ptr(out), h, s, off, _ptr(off_t), prefix_len, 1.0 / math.sqrt(d) if scale is None else scale,
            int(accumulate), _ptr(workspace), nbytes)
    return out


def kv4_attention_workspace(cache: Kv4Cache, num_heads: int, seq_len: int, accumulate: bool = True) -> int:
    """Bytes of workspace of such a kv4_attention call (may be 0)."""
    key = (num_heads, seq_len, accumulate)
    n = cache._workspaces.get(key)
    if n is None:
        size = ctypes.c_int64(0)
        with torch.cuda.device(cache.device):
            check("hrm_kv4_attention_workspace", LIB.hrm_kv4_attention_workspace(cache._ref, num_heads, seq_len,
                                                                                 int(accumulate), ctypes.byref(size)))
        n = cache._workspaces[key] = size.value
    return n


def kv4_evict(cache: Kv4Cache, lengths: Offset, budget: int, protect_from: Offset, out: Optional[Kv4Cache] = None,
              new_lengths: Optional[torch.Tensor] = None, *, stream=None) -> torch.Tensor:
    """Keeps the `budget` rows of largest weight of each kv head; returns the new lengths (int32 [b]).

    lengths: the rows in use; rows whose position is at or past protect_from rank
    above every weight.  In place, or into `out`, another tracked cache of at
    least `budget` rows.  Kept rows below budget stay where they are, the others
    fill the freed places in order.
    """
    to = cache if out is None else out
    b, h, n, d = cache.shape
    if cache.weights is None or cache.positions is None or to.weights is None or to.positions is None:
        raise ValueError("kv4_evict needs caches with weights and positions (kv4_cache(..., track=True))")
    if (to.shape[0], to.shape[1], to.shape[3]) != (b, h, d):
        raise ValueError("out differs from the cache in batch, kv_heads or head_dim")
    length, length_t = _offset(lengths, "lengths", b)
    protect, protect_t = _offset(protect_from, "protect_from", b)
    if new_lengths is None:
        new_lengths = _made(stream, cache.positions.new_empty, b)
    else:
        _need(new_lengths, "new_lengths", (torch.int32,))
        if new_lengths.numel() != b:
            raise ValueError("new_lengths must have one value per sequence")
    _launch("hrm_kv4_evict", cache.device, (to.k_codes, length_t, protect_t, new_lengths), stream, cache._ref, to._ref,
            length, _ptr(length_t), budget, protect, _ptr(protect_t), _ptr(new_lengths))
    return new_lengths
