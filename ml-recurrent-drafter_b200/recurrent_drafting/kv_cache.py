"""Pre-allocated KV cache with the reference's API (recurrent_drafting/kv_cache.py).

One tensor [n_layers, 2, batch, n_kv_heads, max_length, head_dim].  The reference keeps every row
right-aligned and shifts whole rows after each decode step; here a row stays where the prompt put
it and only grows: row b occupies slots [kv_begin[b], kv_begin[b] + kv_len[b]).  kv_begin / kv_len
are device int32 vectors owned by the decode loop; the View/Cache surface below keeps the
reference's scalar `length` semantics for callers that use the cache the reference's way.
"""
from dataclasses import dataclass
from typing import Dict, List, NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _lib


class View:
    """Key or value cache of one layer (kv_cache.py:10-35)."""

    def __init__(self, cache: torch.Tensor, layer: int, kv: int):
        self._cache = cache
        self._layer = layer
        self._kv = kv
        self.length = 0

    @property
    def shape(self) -> Tuple[int, int, int, int]:
        _, _, batch_size, n_heads, _, head_dim = self._cache.shape
        return (batch_size, n_heads, self.length, head_dim)

    @property
    def plane(self) -> torch.Tensor:
        """[batch, n_kv_heads, max_length, head_dim] storage of this view."""
        return self._cache[self._layer, self._kv]

    def cat(self, new_kv: torch.Tensor) -> torch.Tensor:
        _, _, batch_size, n_heads, max_length, head_dim = self._cache.shape
        n = new_kv.shape[2]
        assert new_kv.shape == (batch_size, n_heads, n, head_dim)
        assert self.length + n <= max_length
        self.plane[:, :, self.length : self.length + n, :] = new_kv
        self.length += n
        return self.plane[:, :, : self.length, :]

    def slice(self, prev: int) -> torch.Tensor:
        return self.plane[:, :, prev : self.length, :]


class Cache:
    """kv_cache.py:38-98."""

    def __init__(self, batch_size: int, max_length: int, n_layers: int, n_heads: int, head_dim: int,
                 dtype: torch.dtype, device: torch.device) -> None:
        self._cache = torch.zeros([n_layers, 2, batch_size, n_heads, max_length, head_dim], dtype=dtype, device=device)
        self.sliced = tuple((View(self._cache, layer, 0), View(self._cache, layer, 1)) for layer in range(n_layers))

    @property
    def storage(self) -> torch.Tensor:
        """What the model's backbone() takes."""
        return self._cache

    @property
    def max_length(self) -> int:
        return self._cache.shape[4]

    def set_length(self, length: int) -> None:
        for k, v in self.sliced:
            k.length = v.length = length

    def unpack(self, prompt_length: int, tree_attn_index: torch.Tensor) -> None:
        """Replicates the packed-tree K/V into per-beam layout (kv_cache.py:58-98).  The decode loop
        of this package does not need it (its commit reads the packed slots directly)."""
        batch_size = tree_attn_index.shape[0]
        n_flat = tree_attn_index.shape[1] * tree_attn_index.shape[2]
        n_layers, _, cache_batch, n_heads, max_length, head_dim = self._cache.shape
        idx = tree_attn_index.reshape(batch_size, n_flat).to(torch.int64)
        if batch_size != cache_batch:
            idx = idx.expand(cache_batch, n_flat)
        idx = idx.contiguous()
        scratch = torch.empty([n_layers, 2, cache_batch, n_heads, n_flat, head_dim], dtype=self._cache.dtype,
                              device=self._cache.device)
        _lib.call("rd_cache_unpack", _lib.dtype_code(self._cache.dtype), _lib.ptr(self._cache), n_layers, cache_batch,
                  n_heads, max_length, head_dim, prompt_length, _lib.ptr(idx), n_flat, _lib.ptr(scratch), _lib.stream())
        for k, v in self.sliced:
            k.length = v.length = prompt_length + n_flat

    def unpack_static(self, prompt_length: int, tree_attn_index: torch.Tensor) -> None:
        """Cache.unpack for callers that must not allocate device memory (a host that owns all of the
        device's memory in its own arena, or a loop that forbids allocation after set-up): the staging
        copy lives in a fixed 16 MiB array inside the library instead of a fresh tensor.

        tree_attn_index must already be a contiguous int64 tensor of shape (cache batch, W, Lb) on the
        cache's device, so that this wrapper creates no tensor either.  Raises if the gathered rows
        (n_layers*2*batch*heads*W*Lb*head_dim elements) do not fit; calls that can overlap on the GPU
        share the array and must be ordered on one stream; make the first call per device at set-up.
        """
        n_layers, _, cache_batch, n_heads, max_length, head_dim = self._cache.shape
        idx = tree_attn_index
        assert idx.dtype == torch.int64 and idx.is_contiguous() and idx.shape[0] == cache_batch
        n_flat = idx.shape[1] * idx.shape[2]
        _lib.call("rd_cache_unpack_static", _lib.dtype_code(self._cache.dtype), _lib.ptr(self._cache), n_layers, cache_batch,
                  n_heads, max_length, head_dim, prompt_length, _lib.ptr(idx), n_flat, _lib.stream())
        for k, v in self.sliced:
            k.length = v.length = prompt_length + n_flat


class LayerCodes(NamedTuple):
    """One layer of a QuantizedCache: codes [batch, heads, capacity, head_dim * bits / 8] (uint8) and parameters [batch, heads, capacity, 2]
    (int16: the bf16 pattern of the scale, zero)."""

    k_codes: torch.Tensor
    k_params: torch.Tensor
    v_codes: torch.Tensor
    v_params: torch.Tensor


class QuantizedCache:
    """Keys and values in codes of 8 or 4 bits, with a scale and a zero for each token of a head: a half or a quarter of a bf16 cache's
    memory, and of the bytes that attention reads.  Rows are quantised as they are written (append), read back in a plain type (read), and
    attended to where they lie (attend); slots and rows as in Cache.  A code stands for scale * (code - zero), zero being exact; see
    rd_cache_quant_append in include/redrafter_b200.h for the rounding.

    A row of batch, head and slot holds its values alone, so a slot may be written again at any time, and what lies past a row's length
    is never looked at."""

    SLOTS = 64  # the storage has a multiple of these

    def __init__(self, batch_size: int, max_length: int, n_layers: int, n_heads: int, head_dim: int, bits: int, device) -> None:
        if bits not in (4, 8):
            raise _lib.RedrafterError(f"a cache is held in 4 or 8 bits, not in {bits}")
        if head_dim % 8 or not 8 <= head_dim <= 256:
            raise _lib.RedrafterError(f"heads of {head_dim} features: a multiple of 8 up to 256 is wanted")
        self.bits, self.head_dim, self.max_length, self.length = bits, head_dim, max_length, 0
        capacity = (max_length + self.SLOTS - 1) // self.SLOTS * self.SLOTS
        self._codes = torch.zeros(n_layers, 2, batch_size, n_heads, capacity, head_dim * bits // 8, dtype=torch.uint8, device=device)
        self._params = torch.zeros(n_layers, 2, batch_size, n_heads, capacity, 2, dtype=torch.int16, device=device)
        self._shape = (batch_size, n_heads, capacity, head_dim)
        self._workspace_bytes: Dict[Tuple, int] = {}
        self._describe()

    def _describe(self) -> None:
        """What every call needs of the storage: layers, addresses, device."""
        self.layers = [LayerCodes(c[0], p[0], c[1], p[1]) for c, p in zip(self._codes, self._params)]
        self._planes = [tuple(t.data_ptr() for t in l) for l in self.layers]
        self._device: int = self._codes.get_device()

    # copies (copy.deepcopy, pickle) have storage, and so addresses, of their own
    def __getstate__(self) -> Dict:
        return {k: v for k, v in self.__dict__.items() if k not in ("layers", "_planes", "_device")}

    def __setstate__(self, state: Dict) -> None:
        self.__dict__.update(state)
        self._describe()

    @property
    def storage(self) -> "QuantizedCache":
        """What the model's backbone() takes."""
        return self

    def set_length(self, length: int) -> None:
        self.length = length

    def bytes_per_token(self) -> int:
        n_layers, _, _, heads, _, row = self._codes.shape
        return 2 * n_layers * heads * (row + 4)

    def _on_device(self) -> int:
        """The cache's device, which has to be the current one: kernels are launched on its current stream."""
        if self._device < 0:
            raise _lib.RedrafterError("operator called with a CPU tensor: this library has no CPU path")
        if self._device != torch._C._cuda_getDevice():
            raise _lib.RedrafterError(f"the cache lies on cuda:{self._device}, which is not the current device")
        return self._device

    def _elsewhere(self, **tensors) -> None:
        for name, t in tensors.items():
            if t is not None and t.get_device() != self._device:
                raise _lib.RedrafterError(f"{name} lies on {t.device}, the cache on cuda:{self._device}")

    def _index(self, name: str, t: torch.Tensor, n: int) -> int:
        """The address of a vector of indices."""
        if t.dtype is not torch.int32 or t.numel() < n or t.dim() != 1 or not t.is_contiguous():
            raise _lib.RedrafterError(f"{name} is a contiguous int32 vector of {n} elements")
        if t.get_device() != self._device:
            self._elsewhere(**{name: t})
        return t.data_ptr()

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, tok_row: torch.Tensor, tok_slot: torch.Tensor,
               m_dev: Optional[torch.Tensor] = None) -> None:
        """Writes the keys and values [tokens, heads, head_dim] of new tokens (bf16 or fp32; tokens and heads any multiples of 16 bytes
        apart, the same in both) to slots tok_slot of batch rows tok_row.  Two tokens must not have the same place."""
        B, heads, capacity, hd = self._shape
        dims = k.shape
        if len(dims) != 3 or dims[1] != heads or dims[2] != hd or v.shape != dims or k.dtype is not v.dtype:
            raise _lib.RedrafterError(f"keys {tuple(k.shape)} and values {tuple(v.shape)}: [tokens, {heads}, {hd}] of one type is wanted")
        m = dims[0]
        # the stride of a dimension of size 1 says nothing
        s, u = k.stride(), v.stride()
        tok, head = (s[0] if m > 1 else 0), (s[1] if heads > 1 else 0)
        if s[2] != 1 or u[2] != 1 or (m > 1 and u[0] != tok) or (heads > 1 and u[1] != head):
            raise _lib.RedrafterError("keys and values need the same strides, and their features one after another")
        if m_dev is not None and (m_dev.dtype is not torch.int32 or m_dev.numel() < 1):
            raise _lib.RedrafterError("m_dev is an int32 count")
        dev = self._on_device()
        if k.get_device() != dev or v.get_device() != dev or (m_dev is not None and m_dev.get_device() != dev):
            self._elsewhere(k=k, v=v, m_dev=m_dev)
        rows, slots = self._index("tok_row", tok_row, m), self._index("tok_slot", tok_slot, m)
        _lib.call("rd_cache_quant_append", _lib.CACHE_APPEND.pack(
            k.data_ptr(), v.data_ptr(), tok, head, *self._planes[layer], rows, slots, 0 if m_dev is None else m_dev.data_ptr(),
            _lib.dtype_code(k.dtype), self.bits, m, B, heads, hd, capacity), _lib.stream())

    def read(self, layer: int, begin: torch.Tensor, length: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor) -> None:
        """Slots begin[b] .. begin[b] + length[b] - 1 of every row b as plain keys and values: rows 0 .. of k_out and v_out [batch, heads,
        rows, head_dim] (bf16 or fp32, contiguous).  What lies behind a row's last is left as it was."""
        B, heads, capacity, hd = self._shape
        dims = k_out.shape
        if len(dims) != 4 or dims[0] != B or dims[1] != heads or dims[3] != hd or v_out.shape != dims or k_out.dtype is not v_out.dtype:
            raise _lib.RedrafterError(f"outputs {tuple(k_out.shape)} and {tuple(v_out.shape)}: [{B}, {heads}, rows, {hd}] of one type is wanted")
        if not (k_out.is_contiguous() and v_out.is_contiguous()):
            raise _lib.RedrafterError("the outputs are contiguous")
        dev = self._on_device()
        if k_out.get_device() != dev or v_out.get_device() != dev:
            self._elsewhere(k_out=k_out, v_out=v_out)
        first, count = self._index("begin", begin, B), self._index("length", length, B)
        _lib.call("rd_cache_quant_read", _lib.CACHE_READ.pack(*self._planes[layer], first, count, k_out.data_ptr(), v_out.data_ptr(),
                                                              _lib.dtype_code(k_out.dtype), self.bits, B, heads, hd, capacity, dims[2]), _lib.stream())

    def attend(self, layer: int, q: torch.Tensor, out: torch.Tensor, row_start: torch.Tensor, kv_begin: torch.Tensor, base_len: torch.Tensor,
               max_new: int, max_kv: int, mode: int = _lib.ATTN_CAUSAL, tree_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
               status: Optional[torch.Tensor] = None) -> None:
        """Attention of new tokens, whose keys and values have been appended.  q [tokens, query heads * head_dim] (bf16 or fp32; rows any
        multiple of 16 bytes apart), out the same, contiguous; row b of the batch has tokens row_start[b] .. row_start[b + 1] - 1, its keys are slots
        kv_begin[b] .. + base_len[b] (all visible) and its new tokens' own, visible causally or through tree_mask [tokens, words] (ATTN_TREE).
        max_new, max_kv: upper bounds of a row's new tokens and keys; what exceeds them is left out.  scale: of the scores, 1 / sqrt(head_dim) unless
        given."""
        B, heads, capacity, hd = self._shape
        dims = q.shape
        if len(dims) != 2 or dims[1] == 0 or dims[1] % (heads * hd) or out.shape != dims or out.dtype is not q.dtype or not out.is_contiguous():
            raise _lib.RedrafterError(f"queries {tuple(q.shape)}, output {tuple(out.shape)}: [tokens, a multiple of {heads} heads * {hd}] of one type is wanted")
        m, width = dims
        ldq, step = q.stride()
        if step != 1:
            raise _lib.RedrafterError("the features of a query lie one after another")
        if status is not None and (status.dtype is not torch.int32 or status.numel() < 1):
            raise _lib.RedrafterError("status is an int32 number")
        dev = self._on_device()
        if q.get_device() != dev or out.get_device() != dev or (status is not None and status.get_device() != dev):
            self._elsewhere(q=q, out=out, status=status)
        starts, begins, bases = self._index("row_start", row_start, B + 1), self._index("kv_begin", kv_begin, B), self._index("base_len", base_len, B)
        words = mask = 0
        if mode == _lib.ATTN_TREE:
            if tree_mask is None or tree_mask.dtype is not torch.int32 or tree_mask.dim() != 2 or tree_mask.shape[0] < m or not tree_mask.is_contiguous():
                raise _lib.RedrafterError("tree_mask is a contiguous int32 matrix with a row for each token")
            self._elsewhere(tree_mask=tree_mask)
            words, mask = tree_mask.shape[1], tree_mask.data_ptr()
        code, nh = _lib.dtype_code(q.dtype), width // hd
        sizes = (code, m, nh, max_new, max_kv)
        need = self._workspace_bytes.get(sizes)
        if need is None:
            need = _lib.load().rd_attention_quant_workspace_bytes(code, self.bits, m, B, nh, heads, hd, max_new, max_kv)
            if len(self._workspace_bytes) >= 256:
                self._workspace_bytes.clear()
            self._workspace_bytes[sizes] = need
        # a new one for each call: calls on other streams and captured graphs each have their own
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
        _lib.call("rd_attention_quant", _lib.ATTENTION_QUANT.pack(
            q.data_ptr(), ldq if m > 1 else width, *self._planes[layer], out.data_ptr(), starts, begins, bases, mask,
            0 if workspace is None else workspace.data_ptr(), max(need, 0), 0 if status is None else status.data_ptr(),
            code, self.bits, m, B, nh, heads, hd, capacity, max_new, max_kv, mode, words, hd ** -0.5 if scale is None else scale), _lib.stream())
        if need > 0:
            _lib.launches += 1  # shares of keys are summed by a kernel of their own

    def commit_draft(self, fp, n_accepted: torch.Tensor, seq_in_beam: torch.Tensor, beam_shape, kv_begin: torch.Tensor) -> None:
        """Moves the accepted tokens of a packed draft behind the rows' prefixes, in all layers."""
        n_layers, _, B, heads, capacity, _ = self._codes.shape
        W, L = beam_shape.width, beam_shape.length
        unpacker = fp.unpacker
        if unpacker.dtype is not torch.int32 or unpacker.numel() < B * W * L or not unpacker.is_contiguous():
            raise _lib.RedrafterError(f"unpacker is a contiguous int32 tensor of {B} * {W} * {L} elements")
        if unpacker.get_device() != self._device:
            self._elsewhere(unpacker=unpacker)
        begin, base, accepted, seq = (self._index(name, t, B) for name, t in (("kv_begin", kv_begin), ("base_len", fp.base_len),
                                                                             ("n_accepted", n_accepted), ("seq_in_beam", seq_in_beam)))
        self._on_device()
        _lib.call("rd_cache_quant_commit", self.bits, self._codes.data_ptr(), self._params.data_ptr(), 2 * n_layers, B, heads, capacity, self.head_dim,
                  begin, base, unpacker.data_ptr(), W, L, accepted, seq, _lib.stream())


@dataclass(frozen=True)
class KeyValueSpec:
    """A layer that keeps keys and values of every token."""

    heads: int
    dim: int
    vdim: int


@dataclass(frozen=True)
class MatrixStateSpec:
    """A layer that keeps a matrix state of fixed size: S [heads, dim, vdim], n [heads, dim], m [heads], fp32."""

    heads: int
    dim: int
    vdim: int


@dataclass(frozen=True)
class LatentSpec:
    """A layer that keeps one vector of every token, from which all heads' keys and values are formed."""

    width: int


LayerSpec = Union[KeyValueSpec, MatrixStateSpec, LatentSpec]


class LayerKeyValues:
    def __init__(self, spec: KeyValueSpec, batch: int, max_length: int, dtype: torch.dtype, device):
        self.keys = torch.zeros(batch, spec.heads, max_length, spec.dim, dtype=dtype, device=device)
        self.values = torch.zeros(batch, spec.heads, max_length, spec.vdim, dtype=dtype, device=device)


class LayerMatrixState:
    def __init__(self, spec: MatrixStateSpec, batch: int, draft_tokens: int, dtype: torch.dtype, device):
        f32 = dict(dtype=torch.float32, device=device)
        self.S = torch.zeros(batch, spec.heads, spec.dim, spec.vdim, **f32)
        self.n = torch.zeros(batch, spec.heads, spec.dim, **f32)
        self.m = torch.zeros(batch, spec.heads, **f32)
        # Projections and gates of the packed draft tokens: a verify step leaves the state alone, and the commit runs the
        # accepted path through the recurrence from here.
        width = 2 * spec.heads * (spec.dim + spec.vdim)
        self.draft_proj = torch.empty(draft_tokens, (width + 31) // 32 * 32, dtype=dtype, device=device) if draft_tokens else None
        self.draft_gates = torch.empty(draft_tokens, 2 * spec.heads, **f32) if draft_tokens else None


class LayerLatents:
    def __init__(self, spec: LatentSpec, batch: int, max_length: int, dtype: torch.dtype, device):
        self.rows = torch.zeros(batch, 1, max_length, spec.width, dtype=dtype, device=device)


class HybridCache:
    """State of a decoder whose layers differ in what they carry from token to token.  Attention layers keep keys
    [batch, heads, max_length, dim] and values [batch, heads, max_length, vdim], or latents [batch, 1, max_length, width],
    slot = position in the row; recurrent layers keep their state.  Rows are independent; a row whose length is 0 starts afresh whatever its memory holds (the
    recurrent kernels take the zero state then, and no key beyond a row's length is ever read), so giving a row back is
    setting its length to 0."""

    def __init__(self, layers: Sequence[LayerSpec], batch_size: int, max_length: int, dtype: torch.dtype, device,
                 draft_tokens: int = 0) -> None:
        self.max_length = max_length
        self.batch_size = batch_size
        self.length = 0
        self.layers: List[Union[LayerKeyValues, LayerMatrixState, LayerLatents]] = []
        for spec in layers:
            if isinstance(spec, KeyValueSpec):
                self.layers.append(LayerKeyValues(spec, batch_size, max_length, dtype, device))
            elif isinstance(spec, MatrixStateSpec):
                self.layers.append(LayerMatrixState(spec, batch_size, draft_tokens, dtype, device))
            elif isinstance(spec, LatentSpec):
                self.layers.append(LayerLatents(spec, batch_size, max_length, dtype, device))
            else:
                raise TypeError(f"unknown layer spec {spec!r}")

    @property
    def storage(self) -> "HybridCache":
        return self

    def set_length(self, length: int) -> None:
        self.length = length

    def bytes_per_token(self) -> int:
        """Memory that grows with the sequence."""
        planes = [p for l in self.layers for p in ((l.keys, l.values) if isinstance(l, LayerKeyValues) else
                                                   (l.rows,) if isinstance(l, LayerLatents) else ())]
        return sum(p[0, :, 0].numel() * p.element_size() for p in planes)
