"""Torch-facing wrapper of the 8-bit KV cache (include/clove_fp8.h): the
counterpart of ops.KVPool whose cache holds e4m3 codes with one scale per
(block of tokens, KV head).

  codes         float8_e4m3fn [2, num_blocks, num_kv_heads, block_size, head_dim]
  scales        float32 [2, num_blocks, num_kv_heads]; an element is code * scale
  mass          float32 [num_blocks, num_kv_heads, block_size]: the attention
                weight a cached token has received (optional)
  block_tables  int32 [batch, max_blocks_per_seq]
  context_lens  int32 [batch]
  q, k, v       float32, bfloat16 or float16
  out           float32 [batch, num_q_heads, head_dim]

No counterpart in the reference, whose kv_cache is f32 (src/nn.rs:534).
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from .ops import _DTYPES, _ptr


# The current stream's handle without a Stream object, where torch offers it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _current_stream(device: int) -> int:
    return _raw_stream(device) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


# The C side takes 32 bits, to which ctypes would cut a larger number down.
_INT_MAX = 2 ** 31 - 1


def _fits(n: int) -> bool:
    return -_INT_MAX <= n <= _INT_MAX


class Fp8KVPool:
    """A paged 8-bit KV cache on one GPU.  `storage`, `scales` and `mass` wrap
    the caller's tensors; what is missing is allocated (mass only with
    track_mass).  Blocks are filled from row 0 on: a write to row 0 starts a
    block anew, whatever an earlier sequence left in it.  A token written to a
    block may rewrite its other rows (to a grown scale): no other sequence or
    call may read a block while it is appended to.

    Scratch comes from the caching allocator call by call, so calls on
    different streams, and graphs captured from them, share none."""

    def __init__(self, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                 device: int | torch.device = 0, storage: torch.Tensor | None = None,
                 scales: torch.Tensor | None = None, mass: torch.Tensor | None = None, track_mass: bool = False):
        self.device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("Fp8KVPool lives on a CUDA device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        shapes = {"storage": ((2, num_blocks, num_kv_heads, block_size, head_dim), torch.float8_e4m3fn),
                  "scales": ((2, num_blocks, num_kv_heads), torch.float32),
                  "mass": ((num_blocks, num_kv_heads, block_size), torch.float32)}
        for name, t in (("storage", storage), ("scales", scales), ("mass", mass)):
            shape, dtype = shapes[name]
            if t is not None and (tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous()
                                  or t.device != self.device):
                raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on {self.device}")
        if (storage is None) != (scales is None):
            raise ValueError("storage and scales go together")
        if storage is None:
            storage = torch.zeros(shapes["storage"][0], dtype=torch.uint8, device=self.device).view(torch.float8_e4m3fn)
            scales = torch.zeros(shapes["scales"][0], dtype=torch.float32, device=self.device)
        if mass is None and track_mass:
            mass = torch.zeros(shapes["mass"][0], dtype=torch.float32, device=self.device)
        self.storage, self.scales, self.mass = storage, scales, mass
        self.num_blocks, self.block_size = num_blocks, block_size
        self.num_kv_heads, self.head_dim = num_kv_heads, head_dim
        self._lib = _lib.lib()
        h = C.c_void_p()
        _lib.check(self._lib.clove_fp8_pool_wrap(self.device.index, _ptr(storage), _ptr(scales), _ptr(mass),
                                                 num_blocks, block_size, num_kv_heads, head_dim, C.byref(h)))
        self.handle = h
        self._sizes: dict[tuple, int] = {}  # scratch bytes by call sizes

    def close(self) -> None:
        if getattr(self, "handle", None):
            self._lib.clove_fp8_pool_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- checks ------------------------------------------------------------
    def _on(self, fn, stream: torch.cuda.Stream | None):
        """fn(stream handle) with the pool's device, and `stream` if one is
        given, current: what fn allocates or copies then belongs to it."""
        if stream is None and torch.cuda.current_device() == self.device.index:
            return fn(_current_stream(self.device.index))
        if stream is not None and stream.device != self.device:
            raise ValueError(f"stream is on {stream.device}, the pool on {self.device}")
        s = stream if stream is not None else torch.cuda.current_stream(self.device)
        with torch.cuda.stream(s):
            return fn(s.cuda_stream)

    def _rows(self, t: torch.Tensor, rows: int, heads: int, name: str, dtype: torch.dtype | None = None) -> torch.Tensor:
        if t.dtype not in _DTYPES or (dtype is not None and t.dtype != dtype) or t.device != self.device:
            want = dtype if dtype is not None else "float32, bfloat16 or float16"
            raise ValueError(f"{name} must be a {want} tensor on {self.device}")
        if t.shape != (rows, heads, self.head_dim):
            if t.numel() != rows * heads * self.head_dim:
                raise ValueError(f"{name} must hold {rows} x {heads} x {self.head_dim} elements, not {tuple(t.shape)}")
            t = t.reshape(rows, heads, self.head_dim)
        if not t.is_contiguous():
            t = t.contiguous()
        return t if t.data_ptr() % 16 == 0 else t.clone()

    def _i32(self, t: torch.Tensor, name: str, dim: int, rows: int | None = None) -> None:
        if t.dtype != torch.int32 or t.device != self.device or t.dim() != dim or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {dim}-D int32 tensor on {self.device}")
        if rows is not None and t.shape[0] != rows:
            raise ValueError(f"{name} has {t.shape[0]} rows, not {rows}")

    def _scratch(self, fn, *args: int) -> tuple[torch.Tensor | None, int, int]:
        """(tensor to hold on to, its address, bytes) of the scratch that a
        call with these sizes needs."""
        n = self._sizes.get((fn.__name__, *args))
        if n is None:
            if len(self._sizes) > 4096:
                self._sizes.clear()
            n = self._sizes[(fn.__name__, *args)] = int(fn(self.handle, *args))
        if n == 0:
            return None, 0, 0
        ws = torch.empty(n, dtype=torch.uint8, device=self.device)
        return ws, ws.data_ptr(), n

    @staticmethod
    def _longest(context_lens: torch.Tensor, extra: int) -> int:
        # forces a device sync; pass max_ctx on hot paths
        return int(context_lens.max().item()) + extra if context_lens.numel() else 0

    # ---- ops ---------------------------------------------------------------
    def reshape_and_cache(self, k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor,
                          stream: torch.cuda.Stream | None = None) -> None:
        """Quantise k, v [num_tokens, num_kv_heads, head_dim] into the slots
        slot_mapping (int32 [num_tokens]; negative: padding, skipped).  A
        block's scale grows to cover what is written and the rows already in
        it are rounded to it; a write to row 0 starts the block anew."""
        self._i32(slot_mapping, "slot_mapping", 1)
        n = slot_mapping.numel()

        def call(s: int) -> int:
            kr = self._rows(k, n, self.num_kv_heads, "k")
            vr = self._rows(v, n, self.num_kv_heads, "v", kr.dtype)
            ws, at, size = self._scratch(self._lib.clove_fp8_append_workspace_size, n)
            return self._lib.clove_fp8_append(self.handle, _DTYPES[kr.dtype], kr.data_ptr(), vr.data_ptr(),
                                              slot_mapping.data_ptr(), n, at, size, s)

        _lib.check(self._on(call, stream))

    def gather_kv(self, block_tables: torch.Tensor, context_lens: torch.Tensor, max_ctx: int,
                  stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The cached tokens as float32 [batch, max_ctx, num_kv_heads,
        head_dim]; rows behind a sequence's last token are zero."""
        self._i32(context_lens, "context_lens", 1)
        b = context_lens.numel()
        self._i32(block_tables, "block_tables", 2, b)
        if not _fits(max_ctx):
            raise ValueError(f"max_ctx {max_ctx} is beyond 32 bits")

        def call(s: int) -> tuple[torch.Tensor, torch.Tensor]:
            shape = (b, max_ctx, self.num_kv_heads, self.head_dim)
            ko = torch.empty(shape, dtype=torch.float32, device=self.device)
            vo = torch.empty(shape, dtype=torch.float32, device=self.device)
            _lib.check(self._lib.clove_fp8_gather(self.handle, _ptr(block_tables), block_tables.shape[1],
                                                  _ptr(context_lens), b, max_ctx, _ptr(ko), _ptr(vo), s))
            return ko, vo

        return self._on(call, stream)

    def decode(self, q: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
               scale: float | None = None, max_ctx: int | None = None, out: torch.Tensor | None = None,
               k_new: torch.Tensor | None = None, v_new: torch.Tensor | None = None, softcap: float = 0.0,
               alibi_slopes: torch.Tensor | None = None, window: int = 0, accumulate: bool = False,
               stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """Decode over the cache; with k_new/v_new the new token is appended
        first (context_lens are then the lengths before it, max_ctx bounds
        those after it).  Scores, in this order: softcap * tanh(. / softcap);
        + alibi_slopes[hq] * (t - (L - 1)) with float32 [num_q_heads] slopes;
        only the last `window` tokens.  accumulate adds each token's weight,
        summed over its KV head's query heads, to the pool's mass."""
        self._i32(context_lens, "context_lens", 1)
        batch = context_lens.shape[0]
        self._i32(block_tables, "block_tables", 2, batch)
        hq = q.shape[1] // self.head_dim if q.dim() == 2 else q.shape[1]
        append = k_new is not None
        if append != (v_new is not None):
            raise ValueError("k_new and v_new go together")
        if alibi_slopes is not None and (alibi_slopes.shape != (hq,) or alibi_slopes.dtype != torch.float32
                                         or alibi_slopes.device != self.device or not alibi_slopes.is_contiguous()):
            raise ValueError(f"alibi_slopes must be a contiguous float32 [{hq}] tensor on {self.device}")
        if softcap and abs(softcap) < torch.finfo(torch.float32).tiny:  # float32 would make it 0, which is no cap
            raise ValueError(f"softcap {softcap} is below float32's range")
        if accumulate and self.mass is None:
            raise ValueError("accumulate needs a pool with mass (track_mass=True)")
        shape = (batch, hq, self.head_dim)
        if out is not None and (out.shape != shape or out.dtype != torch.float32 or out.device != self.device
                                or not out.is_contiguous()):
            raise ValueError(f"out must be a contiguous float32 tensor of shape {shape} on {self.device}")
        if max_ctx is None:
            max_ctx = self._longest(context_lens, int(append))
        if window > _INT_MAX:
            window = _INT_MAX  # longer than any sequence either way
        if not (_fits(max_ctx) and _fits(window)):
            raise ValueError(f"max_ctx {max_ctx}, window {window}: beyond 32 bits")
        if scale is None:
            scale = 1.0 / math.sqrt(self.head_dim)

        def call(s: int) -> torch.Tensor:
            qr = self._rows(q, batch, hq, "q")
            kr = vr = None
            if append:
                kr = self._rows(k_new, batch, self.num_kv_heads, "k_new", qr.dtype)
                vr = self._rows(v_new, batch, self.num_kv_heads, "v_new", qr.dtype)
            o = torch.empty(shape, dtype=torch.float32, device=self.device) if out is None else out
            scores = None
            if softcap or alibi_slopes is not None or window or accumulate:
                scores = C.byref(_lib.Fp8Scores(softcap, _ptr(alibi_slopes), window, bool(accumulate)))
            ws, at, size = self._scratch(self._lib.clove_fp8_decode_workspace_size, batch, hq, max_ctx, bool(accumulate))
            _lib.check(self._lib.clove_fp8_decode(
                self.handle, _DTYPES[qr.dtype], qr.data_ptr(), _ptr(kr), _ptr(vr), hq, block_tables.data_ptr(),
                block_tables.shape[1], context_lens.data_ptr(), batch, scale, max_ctx, scores, o.data_ptr(), at, size, s))
            return o

        return self._on(call, stream)

    def append_decode(self, q, k_new, v_new, block_tables, context_lens, **kw) -> torch.Tensor:
        return self.decode(q, block_tables, context_lens, k_new=k_new, v_new=v_new, **kw)

    def evict(self, block_tables: torch.Tensor, context_lens: torch.Tensor, new_tables: torch.Tensor, budget: int,
              recent: int = 0, max_ctx: int | None = None,
              stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Bring every sequence down to min(context_lens, budget) tokens: each
        KV head keeps the last `recent` ones and the heaviest others (mass;
        ties to the lower index; tokens that no accumulating decode has seen
        have mass 0, a fresh prompt's too), moved in order to the blocks new_tables,
        which must be none of the blocks the sequences hold now.  Returns
        (kept int32 [batch, num_kv_heads, budget], -1 behind the last,
        new_lens int32 [batch]).  Token indices are those of the compacted
        cache from then on (windows and distance biases count in them)."""
        self._i32(context_lens, "context_lens", 1)
        batch = context_lens.numel()
        self._i32(block_tables, "block_tables", 2, batch)
        self._i32(new_tables, "new_tables", 2, batch)
        if self.mass is None:
            raise ValueError("evict needs a pool with mass (track_mass=True)")
        if budget < 1 or not 0 <= recent <= budget:
            raise ValueError(f"budget {budget}, recent {recent}: 0 <= recent <= budget, budget >= 1")
        if max_ctx is None:
            max_ctx = self._longest(context_lens, 0)
        if not (_fits(max_ctx) and _fits(budget)):
            raise ValueError(f"max_ctx {max_ctx}, budget {budget}: beyond 32 bits")

        def call(s: int) -> tuple[torch.Tensor, torch.Tensor]:
            kept = torch.empty((batch, self.num_kv_heads, budget), dtype=torch.int32, device=self.device)
            lens = torch.empty(batch, dtype=torch.int32, device=self.device)
            ws, at, size = self._scratch(self._lib.clove_fp8_evict_workspace_size, batch, max_ctx, budget)
            _lib.check(self._lib.clove_fp8_evict(
                self.handle, _ptr(block_tables), block_tables.shape[1], _ptr(context_lens), batch, max_ctx,
                _ptr(new_tables), new_tables.shape[1], budget, recent, _ptr(kept), _ptr(lens), at, size, s))
            return kept, lens

        return self._on(call, stream)

    def copy_blocks(self, src: torch.Tensor, dst: torch.Tensor, stream: torch.cuda.Stream | None = None) -> None:
        """Copy blocks src[i] -> dst[i] (int32 device tensors): the block
        manager's copy-on-write copies."""
        self._i32(src, "src", 1)
        self._i32(dst, "dst", 1, src.numel())
        _lib.check(self._on(lambda s: self._lib.clove_fp8_copy_blocks(self.handle, _ptr(src), _ptr(dst), src.numel(), s),
                            stream))

    def pool_status(self, stream: torch.cuda.Stream | None = None) -> int:
        """Check flags (FLAG_*) that the pool's calls raised since the last
        read; synchronises the stream."""
        flags = C.c_int(0)
        rc = self._on(lambda s: self._lib.clove_fp8_pool_status(self.handle, s, C.byref(flags)), stream)
        if rc not in (_lib.OK, _lib.ERR_DEVICE_CHECK):
            _lib.check(rc)
        return flags.value
