"""Operator-level Python face of the two ppl.nn operators, on torch CUDA tensors.

Names, attributes, input order and error behaviour follow the llm_cuda engine:
  * attributes and defaults: src/ppl/nn/models/onnx/parsers/opmx/parse_multi_head_cache_attention_param.cc:18-45,
    parse_key_value_cache_param.cc:27-48
  * input order and guards: src/ppl/nn/engines/llm_cuda/kernels/opmx/dynamic_batching/
    multi_head_cache_attention_kernel.cc:27-168 and key_value_cache_kernel.cc:26-110
torch is used for device memory and streams only; all arithmetic happens in the CUDA library.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import capi


@dataclass
class KeyValueCacheParam:
    """src/ppl/nn/params/opmx/key_value_cache_param.h:10-18 (num_layer and layer_idx are required)."""
    num_layer: int
    layer_idx: int
    quant_bit: int = 0
    quant_group: int = 8
    num_repeat: int = 1
    cache_mode: int = 0
    cache_layout: int = 0
    page_size: int = 128


@dataclass
class MultiHeadCacheAttentionParam:
    """src/ppl/nn/params/opmx/multi_head_cache_attention_param.h:10-22."""
    num_heads: int
    head_dim: int
    num_layer: int
    layer_idx: int
    num_kv_heads: int = -1  # parser default: num_heads
    is_causal: bool = True
    is_alibi: bool = False
    quant_bit: int = 0
    quant_group: int = 8
    cache_mode: int = 0
    cache_layout: int = 0
    page_size: int = 128

    def __post_init__(self):
        if self.num_kv_heads < 0:
            self.num_kv_heads = self.num_heads


@dataclass
class MultiHeadAttentionParam:
    """src/ppl/nn/params/opmx/multi_head_attention_param.h."""
    num_heads: int
    head_dim: int
    num_kv_heads: int = -1  # parser default: num_heads
    is_causal: bool = True
    is_alibi: bool = False

    def __post_init__(self):
        if self.num_kv_heads < 0:
            self.num_kv_heads = self.num_heads


@dataclass
class RotaryPositionEmbeddingParam:
    """src/ppl/nn/params/opmx/rotary_position_embedding_param.h; scaling_type "" | "linear" | "dynamic"."""
    theta: float = 10000.0
    bypass_key: int = 0
    rotary_dim: int = 0
    max_position_embeddings: int = 2048
    scaling_type: str = ""
    scaling_factor: float = 1.0


@dataclass
class EngineConfig:
    """The knobs of src/ppl/nn/engines/llm_cuda/engine_config.h:30-35 that reach this path."""
    enable_cache_prefill: bool = False
    specify_decoding_attn_split_k: int = 1
    # accepted for compatibility, ignored: there is one decode algorithm here
    enable_decoding_sharemem_mhca: bool = True
    enable_decoding_infinity_mhca: bool = True
    enable_decoding_infinity_gqca: bool = True
    specify_decoding_attn_tpb: int = 0


class OpError(RuntimeError):
    """An operator returned a non-success RetCode; ``name`` is the RetCode's name."""

    def __init__(self, name: str, msg: str):
        super().__init__(f"{name}: {msg}")
        self.name = name


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _require_cuda(**tensors):
    for name, t in tensors.items():
        if t is None:
            raise OpError("RC_NOT_FOUND", f'Input "{name}" is required.')
        if not t.is_cuda:
            raise OpError("RC_INVALID_VALUE", f"{name} must be a CUDA tensor")
        if not t.is_contiguous():
            raise OpError("RC_INVALID_VALUE", f"{name} must be contiguous")


def _mask_arg(attn_mask):
    """The optional attn_mask input as the C ABI wants it; a tensor of zero elements is "absent", as in the
    reference (multi_head_cache_attention_kernel.cc:107)."""
    if attn_mask is None or attn_mask.numel() == 0:
        return None
    _require_cuda(attn_mask=attn_mask)
    if attn_mask.dtype != torch.float16:
        raise OpError("RC_UNSUPPORTED", "attn_mask must be fp16")
    if attn_mask.dim() not in (2, 3):
        raise OpError("RC_INVALID_VALUE", "attn_mask must be [T, C] or [num_heads, T, C]")
    return capi.AttnMask.of(attn_mask.data_ptr(), tuple(attn_mask.shape))


def _max_tokens(cache: torch.Tensor, layout: int) -> int:
    if layout == 0:
        return cache.shape[0]
    if layout == 3:
        return cache.shape[3]
    raise OpError("RC_UNSUPPORTED", "currently only support cache_layout == 0 or cache_layout == 3")


class _Base:
    def __init__(self):
        self.lib = capi.library()

    def _raise(self, fn: str, rc: int):
        if rc != capi.SUCCESS:
            raise OpError(self.lib.status_str(rc), f"{fn} failed")


class MultiHeadCacheAttention(_Base):
    """opmx.dynamic_batching.MultiHeadCacheAttention."""

    def __init__(self, param: MultiHeadCacheAttentionParam, config: EngineConfig | None = None):
        super().__init__()
        self.param = param
        self.config = config or EngineConfig()
        self._workspace: torch.Tensor | None = None

    def make_params(self, *, batch, decoding_batches, max_seqlen, max_kvlen, total_tokens, max_tokens,
                    cachestart_stride_b=0, phase_mask=0) -> capi.AttnParams:
        a, c = self.param, self.config
        p = capi.AttnParams()
        p.num_heads, p.num_kv_heads, p.head_dim = a.num_heads, a.num_kv_heads, a.head_dim
        p.is_causal = int(a.is_causal)
        p.num_layer, p.layer_idx = a.num_layer, a.layer_idx
        p.quant_bit, p.quant_group = a.quant_bit, a.quant_group
        p.cache_mode, p.cache_layout, p.page_size = a.cache_mode, a.cache_layout, a.page_size
        p.enable_cache_prefill = int(c.enable_cache_prefill)
        p.split_k_mode = int(c.specify_decoding_attn_split_k)
        p.phase_mask = phase_mask
        p.batch, p.decoding_batches = batch, decoding_batches
        p.max_seqlen, p.max_kvlen = max_seqlen, max_kvlen
        p.total_tokens, p.max_tokens = total_tokens, max_tokens
        p.cachestart_stride_b = cachestart_stride_b
        self._raise("pplb200_fill_cache_strides", self.lib.fill_cache_strides(p))
        return p

    def workspace_for(self, p: capi.AttnParams, device) -> torch.Tensor:
        rc, nbytes = self.lib.mhca_workspace_size(p)
        self._raise("pplb200_mhca_workspace_size", rc)
        if self._workspace is None or self._workspace.numel() < nbytes or self._workspace.device != device:
            # grow-only scratch, like the engine's tmp-buffer pool (llm_cuda_device.h:151-156)
            self._workspace = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)
        return self._workspace

    def forward(self, query, current_key, current_value, seqstarts, kvstarts, cachestarts, start_pos,
                decoding_batches: int, max_seqlen: int, max_kvlen: int, cache, scale=None, attn_mask=None,
                attn_output: torch.Tensor | None = None, phase_mask: int = 0) -> torch.Tensor:
        a = self.param
        _require_cuda(query=query, current_key=current_key, current_value=current_value, seqstarts=seqstarts,
                      kvstarts=kvstarts, cachestarts=cachestarts, start_pos=start_pos, cache=cache)
        if a.is_alibi:
            raise OpError("RC_UNSUPPORTED", "currently only support is_alibi == false")
        if scale is None or scale.numel() == 0:
            raise OpError("RC_UNSUPPORTED", "currently only support qunatized cache but scale not found")
        mask = _mask_arg(attn_mask)
        _require_cuda(scale=scale)
        stride_b = 0
        if a.cache_mode == 1:
            if cachestarts.dim() != 2:
                raise OpError("RC_INVALID_VALUE", "cachestarts must be a 2d tensor in cache_mode 1")
            stride_b = cachestarts.shape[1]
        batch = start_pos.shape[0]
        p = self.make_params(batch=batch, decoding_batches=int(decoding_batches), max_seqlen=int(max_seqlen),
                             max_kvlen=int(max_kvlen), total_tokens=query.shape[0],
                             max_tokens=_max_tokens(cache, a.cache_layout), cachestart_stride_b=stride_b,
                             phase_mask=phase_mask)
        if attn_output is None:
            attn_output = torch.empty_like(query)
        ws = self.workspace_for(p, query.device)
        if mask is None:
            rc = self.lib.mhca_forward(p, _ptr(query), _ptr(current_key), _ptr(current_value), _ptr(seqstarts),
                                       _ptr(kvstarts), _ptr(cachestarts), _ptr(start_pos), _ptr(cache), _ptr(scale),
                                       _ptr(ws), ws.numel(), _ptr(attn_output), _stream())
        else:
            rc = self.lib.mhca_forward_masked(p, _ptr(query), _ptr(current_key), _ptr(current_value), _ptr(seqstarts),
                                              _ptr(kvstarts), _ptr(cachestarts), _ptr(start_pos), _ptr(cache),
                                              _ptr(scale), mask, _ptr(ws), ws.numel(), _ptr(attn_output), _stream())
        self._raise("pplb200_mhca_forward", rc)
        self._last_params = p
        return attn_output

    def device_status(self) -> int:
        """Status word left by the kernels of the last forward (synchronises the stream)."""
        if self._workspace is None:
            return 0
        rc, s = self.lib.mhca_device_status(_ptr(self._workspace), _stream())
        self._raise("pplb200_mhca_device_status", rc)
        return s


class KeyValueCache(_Base):
    """opmx.dynamic_batching.KeyValueCache: append, then return the dequantised history."""

    def __init__(self, param: KeyValueCacheParam):
        super().__init__()
        self.param = param

    def _params(self, num_kv_heads, head_dim, batch, total_tokens, max_tokens, stride_b) -> capi.AttnParams:
        a = self.param
        p = capi.AttnParams()
        p.num_heads = p.num_kv_heads = num_kv_heads
        p.head_dim = head_dim
        p.is_causal = 1
        p.num_layer, p.layer_idx = a.num_layer, a.layer_idx
        p.quant_bit, p.quant_group = a.quant_bit, a.quant_group
        p.cache_mode, p.cache_layout, p.page_size = a.cache_mode, a.cache_layout, a.page_size
        p.batch, p.total_tokens, p.max_tokens = batch, total_tokens, max_tokens
        p.cachestart_stride_b = stride_b
        self._raise("pplb200_fill_cache_strides", self.lib.fill_cache_strides(p))
        return p

    def forward(self, current_key, current_value, seqstarts, kvstarts, cachestarts, start_pos, max_seqlen: int,
                max_kvlen: int, cache, scale=None, total_kv: int | None = None):
        a = self.param
        _require_cuda(current_key=current_key, current_value=current_value, seqstarts=seqstarts, kvstarts=kvstarts,
                      cachestarts=cachestarts, start_pos=start_pos, cache=cache)
        if scale is None:
            raise OpError("RC_UNSUPPORTED", "currently only support qunatized cache but scale not found")
        if a.num_repeat != 1:
            raise OpError("RC_UNSUPPORTED", "currently only support num_repeat == 1")
        if current_key.dtype != torch.float16:
            raise OpError("RC_UNSUPPORTED", "currently only support fp16")
        _require_cuda(scale=scale)
        stride_b = cachestarts.shape[1] if (a.cache_mode == 1 and cachestarts.dim() == 2) else 0
        if a.cache_mode == 1 and cachestarts.dim() != 2:
            raise OpError("RC_INVALID_VALUE", "cachestarts must be a 2d tensor in cache_mode 1")
        T, Hkv, Dh = current_key.shape
        batch = start_pos.shape[0]
        p = self._params(Hkv, Dh, batch, T, _max_tokens(cache, a.cache_layout), stride_b)
        s = _stream()
        self._raise("pplb200_kv_append_i8g8",
                    self.lib.kv_append(p, _ptr(current_key), _ptr(current_value), _ptr(seqstarts), _ptr(cachestarts),
                                       _ptr(start_pos), _ptr(cache), _ptr(scale), s))
        if total_kv is None:
            # shape inference reads kvstarts[-1] on the host, as the reference op does
            # (ops/opmx/dynamic_batching/key_value_cache_op.cc:37-56)
            total_kv = int(kvstarts[-1].item())
        key = torch.empty((total_kv, Hkv, Dh), dtype=torch.float16, device=current_key.device)
        value = torch.empty_like(key)
        self._raise("pplb200_kv_gather_dequant",
                    self.lib.kv_gather_dequant(p, _ptr(kvstarts), _ptr(cachestarts), _ptr(cache), _ptr(scale),
                                               total_kv, _ptr(key), _ptr(value), s))
        return key, value


class MultiHeadAttention(_Base):
    """opmx.dynamic_batching.MultiHeadAttention: attention over this call's own key/value tensors, no cache
    (src/ppl/nn/engines/llm_cuda/kernels/opmx/dynamic_batching/multi_head_attention_kernel.cc:24-128)."""

    def __init__(self, param: MultiHeadAttentionParam):
        super().__init__()
        self.param = param
        self._workspace: torch.Tensor | None = None

    def forward(self, query, key, value, seqstarts, kvstarts, decoding_batches: int, max_seqlen: int, max_kvlen: int,
                attn_mask=None, attn_output: torch.Tensor | None = None) -> torch.Tensor:
        a = self.param
        _require_cuda(query=query, key=key, value=value, seqstarts=seqstarts, kvstarts=kvstarts)
        if a.is_alibi:
            raise OpError("RC_UNSUPPORTED", "currently only support is_alibi == false")
        mask = _mask_arg(attn_mask)
        p = capi.MhaParams()
        p.num_heads, p.num_kv_heads, p.head_dim, p.is_causal = a.num_heads, a.num_kv_heads, a.head_dim, int(a.is_causal)
        p.batch = seqstarts.shape[0] - 1
        p.decoding_batches = int(decoding_batches)
        p.max_seqlen, p.max_kvlen = int(max_seqlen), int(max_kvlen)
        p.total_tokens, p.total_kv_tokens = query.shape[0], key.shape[0]
        if attn_output is None:
            attn_output = torch.empty_like(query)
        if self._workspace is None or self._workspace.device != query.device:
            self._workspace = torch.empty(256, dtype=torch.uint8, device=query.device)
        rc = self.lib.mha_forward_masked(p, _ptr(query), _ptr(key), _ptr(value), _ptr(seqstarts), _ptr(kvstarts), mask,
                                         _ptr(self._workspace), self._workspace.numel(), _ptr(attn_output), _stream())
        self._raise("pplb200_mha_forward", rc)
        return attn_output

    def device_status(self) -> int:
        if self._workspace is None:
            return 0
        rc, status = self.lib.mhca_device_status(_ptr(self._workspace), _stream())
        self._raise("pplb200_mhca_device_status", rc)
        return status


class RotaryPositionEmbedding(_Base):
    """opmx.dynamic_batching.RotaryPositionEmbedding
    (src/ppl/nn/engines/llm_cuda/kernels/opmx/dynamic_batching/rotary_position_embedding_kernel.cc:24-132),
    and ``forward_fused``: the same rotation fused with the quantise-and-append of the KV cache."""

    _SCALING = {"": 0, "linear": 1, "dynamic": 2}

    def __init__(self, param: RotaryPositionEmbeddingParam):
        super().__init__()
        if param.scaling_type not in self._SCALING:
            raise OpError("RC_UNSUPPORTED", f"unsupported scaling_type: {param.scaling_type}")
        self.param = param
        self._workspace: torch.Tensor | None = None

    def _params(self, query, key, start_pos, max_seqlen) -> capi.RopeParams:
        a = self.param
        p = capi.RopeParams()
        p.num_heads, p.num_kv_heads, p.head_dim = query.shape[1], key.shape[1], query.shape[2]
        p.rotary_dim, p.bypass_key = a.rotary_dim, int(a.bypass_key)
        p.scaling_type = self._SCALING[a.scaling_type]
        p.max_position_embeddings = a.max_position_embeddings
        p.theta, p.scaling_factor = a.theta, a.scaling_factor
        p.batch, p.max_seqlen, p.total_tokens = start_pos.shape[0], int(max_seqlen), query.shape[0]
        return p

    def _ws(self, p, device) -> torch.Tensor:
        rc, nbytes = self.lib.rope_workspace_size(p)
        self._raise("pplb200_rope_workspace_size", rc)
        if self._workspace is None or self._workspace.numel() < nbytes or self._workspace.device != device:
            self._workspace = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)
        return self._workspace

    def forward(self, query, key, seqstarts, start_pos, max_seqlen: int, rotated_query=None, rotated_key=None):
        _require_cuda(query=query, key=key, seqstarts=seqstarts, start_pos=start_pos)
        if query.dtype != torch.float16:
            raise OpError("RC_UNSUPPORTED", "currently only support fp16")
        p = self._params(query, key, start_pos, max_seqlen)
        ws = self._ws(p, query.device)
        rotated_query = torch.empty_like(query) if rotated_query is None else rotated_query
        rotated_key = torch.empty_like(key) if rotated_key is None else rotated_key
        rc = self.lib.rope_forward(p, _ptr(query), _ptr(key), _ptr(seqstarts), _ptr(start_pos), _ptr(ws), ws.numel(),
                                   _ptr(rotated_query), _ptr(rotated_key), _stream())
        self._raise("pplb200_rope_forward", rc)
        return rotated_query, rotated_key

    def forward_fused(self, attn: "MultiHeadCacheAttention", query, key, value, seqstarts, cachestarts, start_pos,
                      max_seqlen: int, cache, scale, want_rotated_key: bool = True):
        """Rotate, then quantise-and-append in the same kernel.  Returns (rotated_query, rotated_key or None);
        follow with ``attn.forward(..., phase_mask=PHASE_DECODE | PHASE_PREFILL)``."""
        _require_cuda(query=query, key=key, value=value, seqstarts=seqstarts, cachestarts=cachestarts,
                      start_pos=start_pos, cache=cache, scale=scale)
        p = self._params(query, key, start_pos, max_seqlen)
        ws = self._ws(p, query.device)
        ap = attn.make_params(batch=start_pos.shape[0], decoding_batches=0, max_seqlen=int(max_seqlen),
                              max_kvlen=0, total_tokens=query.shape[0],
                              max_tokens=_max_tokens(cache, attn.param.cache_layout),
                              cachestart_stride_b=cachestarts.shape[1] if cachestarts.dim() == 2 else 0)
        rotated_query = torch.empty_like(query)
        rotated_key = torch.empty_like(key) if want_rotated_key else None
        rc = self.lib.rope_kv_append(p, ap, _ptr(query), _ptr(key), _ptr(value), _ptr(seqstarts), _ptr(cachestarts),
                                     _ptr(start_pos), _ptr(ws), ws.numel(), _ptr(rotated_query), _ptr(rotated_key),
                                     _ptr(cache), _ptr(scale), _stream())
        self._raise("pplb200_rope_kv_append_i8g8", rc)
        return rotated_query, rotated_key


def _require(device: int, dtype: torch.dtype, **tensors) -> None:
    """Contiguous CUDA tensors of one device (by index) and type."""
    for name, t in tensors.items():
        if t is None or not (t.is_cuda and t.is_contiguous()):
            _require_cuda(**{name: t})
        if t.get_device() != device:
            raise OpError("RC_INVALID_VALUE", f"{name} is on {t.device}, not on cuda:{device}")
        if t.dtype != dtype:
            raise OpError("RC_INVALID_VALUE" if dtype == torch.int64 else "RC_UNSUPPORTED", f"{name} must be {dtype}")


class _CacheOp(_Base):
    """What the operators around the cache share: checks, parameters from the cache's geometry, and a workspace whose
    first word is the device status word.  The workspace is allocated per call, so that calls of one object on two
    streams, or in two captured graphs, never share one; the last call's, and its stream, are kept for
    device_status()."""

    def __init__(self, param):
        super().__init__()
        self.param = param
        self._workspace: torch.Tensor | None = None
        self._call_stream = 0

    def _check_cache(self, cache, scale):
        """(device, kv heads, head_dim, rows) of an INT8 cache with num_layer layers and its scales."""
        if scale is None or scale.numel() == 0:
            raise OpError("RC_UNSUPPORTED", "currently only support qunatized cache but scale not found")
        _require_cuda(cache=cache)
        device = cache.get_device()
        _require(device, torch.int8, cache=cache)
        _require(device, torch.float16, scale=scale)
        return device, *self._cache_shape(tuple(cache.shape), tuple(scale.shape))

    def _cache_shape(self, shape, scale_shape):
        """(kv heads, head_dim, rows) of a cache and its scales."""
        a = self.param
        if len(shape) != 5 or scale_shape != shape[:4] + (shape[4] // 8,):
            raise OpError("RC_INVALID_VALUE", "cache and scale do not belong together")
        if a.cache_layout == 0:
            rows, layers, kv, heads, dim = shape
        elif a.cache_layout == 3:
            layers, kv, heads, rows, dim = shape
        else:
            raise OpError("RC_UNSUPPORTED", "currently only support cache_layout == 0 or cache_layout == 3")
        if layers != a.num_layer or kv != 2:
            raise OpError("RC_INVALID_VALUE", "cache does not have num_layer layers of K and V")
        return heads, dim, rows

    def _check_weight(self, device, weight, heads, rows) -> None:
        _require(device, torch.float32, weight=weight)
        if weight.shape != (self.param.num_layer, heads, rows):
            raise OpError("RC_INVALID_VALUE", "weight must be [num_layer, num_kv_heads, max_tokens]")

    def _params(self, num_heads, num_kv_heads, head_dim, batch, max_kvlen, max_tokens, cachestarts, max_seqlen=0,
                total_tokens=0, is_causal=True) -> capi.AttnParams:
        a = self.param
        if cachestarts.dim() != 1 + (a.cache_mode == 1) or cachestarts.shape[0] != batch:
            raise OpError("RC_INVALID_VALUE", "cachestarts must have an entry (cache_mode 1: a row) per sequence")
        if getattr(a, "num_repeat", 1) != 1:
            raise OpError("RC_UNSUPPORTED", "currently only support num_repeat == 1")
        stride_b = cachestarts.shape[1] if a.cache_mode == 1 else 0
        p = capi.AttnParams(num_heads, num_kv_heads, head_dim, int(is_causal), a.num_layer, a.layer_idx, a.quant_bit,
                            a.quant_group, a.cache_mode, a.cache_layout, a.page_size, 0, 0, 0, batch, 0,
                            int(max_seqlen), int(max_kvlen), total_tokens, max_tokens, 0, 0, 0, 0, stride_b)
        self._raise("pplb200_fill_cache_strides", self.lib.fill_cache_strides(p))
        return p

    def _query_params(self, query, seqstarts, cachestarts, start_pos, max_seqlen, max_kvlen, cache, scale):
        """Checks and parameters of the operators whose query tokens attend to the cache."""
        a = self.param
        device, heads, dim, rows = self._check_cache(cache, scale)
        _require(device, torch.float16, query=query)
        _require(device, torch.int64, seqstarts=seqstarts, cachestarts=cachestarts, start_pos=start_pos)
        if a.is_alibi:
            raise OpError("RC_UNSUPPORTED", "currently only support is_alibi == false")
        if query.shape[1:] != (a.num_heads, a.head_dim) or heads != a.num_kv_heads or dim != a.head_dim:
            raise OpError("RC_INVALID_VALUE", "query or cache does not have the shape of the attributes")
        batch = start_pos.numel()
        if start_pos.dim() != 1 or seqstarts.shape != (batch + 1,):
            raise OpError("RC_INVALID_VALUE", "seqstarts must have one entry more than start_pos")
        return device, self._params(a.num_heads, heads, dim, batch, max_kvlen, rows, cachestarts, max_seqlen,
                                    query.shape[0], a.is_causal)

    def _call(self, name, size_fn, fn, p, device: int, empty: bool, *args) -> None:
        """Runs fn(p, *args, workspace, bytes, stream) on the tensors' device and its current stream.  A call without
        anything to do launches nothing and leaves no status word."""
        if device != torch._C._cuda_getDevice():
            with torch.cuda.device(device):
                return self._call(name, size_fn, fn, p, device, empty, *args)
        rc, nbytes = size_fn(p)
        if empty and rc == capi.SUCCESS:
            self._workspace = None
        elif rc == capi.SUCCESS:
            self._workspace = ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
            # the current stream's handle; a Stream object around it costs 5 us, a fifth of a small call
            self._call_stream = torch._C._cuda_getCurrentRawStream(device)
            rc = fn(p, *args, ws.data_ptr(), nbytes, self._call_stream)
        self._raise(name, rc)

    def device_status(self) -> int:
        """Status word left by the kernels of the last forward.  Synchronises its stream, and the current one: a
        captured forward is replayed there."""
        if self._workspace is None:
            return 0
        with torch.cuda.device(self._workspace.device):
            for stream in dict.fromkeys((self._call_stream, _stream())):
                rc, s = self.lib.mhca_device_status(_ptr(self._workspace), stream)
                self._raise("pplb200_mhca_device_status", rc)
        return s  # the last reading: both streams are done by then


class TreeAttention(_CacheOp):
    """Attention of a tree of drafted tokens over the cache, in which they already are (positions start_pos[b] + i):
    drafted token i sees the history, itself and its ancestors.  ``parents`` [tokens] holds the index, among its
    sequence's drafted tokens, of each one's parent (before it), -1 for a child of the history; None for a chain."""

    def __init__(self, param: MultiHeadCacheAttentionParam):
        super().__init__(param)

    def forward(self, query, parents, seqstarts, cachestarts, start_pos, max_seqlen: int, max_kvlen: int, cache, scale,
                attn_output: torch.Tensor | None = None) -> torch.Tensor:
        device, p = self._query_params(query, seqstarts, cachestarts, start_pos, max_seqlen, max_kvlen, cache, scale)
        if parents is not None:
            _require(device, torch.int64, parents=parents)
            if parents.shape != query.shape[:1]:
                raise OpError("RC_INVALID_VALUE", "parents must have an entry per query token")
        if attn_output is None:
            attn_output = torch.empty_like(query)
        else:
            _require(device, torch.float16, attn_output=attn_output)
            if attn_output.shape != query.shape:
                raise OpError("RC_INVALID_VALUE", "attn_output must be like query")
        self._call("pplb200_tree_attn_forward", self.lib.tree_attn_workspace_size, self.lib.tree_attn_forward, p, device,
                   p.batch == 0 or p.total_tokens == 0, _ptr(query), _ptr(parents), _ptr(seqstarts), _ptr(cachestarts), _ptr(start_pos), _ptr(cache),
                   _ptr(scale), _ptr(attn_output))
        return attn_output


class AttentionWeight(_CacheOp):
    """Adds to ``weight`` [num_layer, num_kv_heads, max_tokens] (fp32, by cache row) the softmax weights that this
    call's query tokens give each cached position, summed over the tokens and the query heads of a kv group.  The
    tokens themselves have been appended already."""

    def __init__(self, param: MultiHeadCacheAttentionParam):
        super().__init__(param)

    def forward(self, query, seqstarts, cachestarts, start_pos, max_seqlen: int, max_kvlen: int, cache, scale,
                weight) -> torch.Tensor:
        device, p = self._query_params(query, seqstarts, cachestarts, start_pos, max_seqlen, max_kvlen, cache, scale)
        self._check_weight(device, weight, p.num_kv_heads, p.max_tokens)
        self._call("pplb200_attn_weight_accumulate", self.lib.attn_weight_workspace_size, self.lib.attn_weight_accumulate,
                   p, device, p.batch == 0 or p.total_tokens == 0, _ptr(query), _ptr(seqstarts), _ptr(cachestarts), _ptr(start_pos), _ptr(cache), _ptr(scale),
                   _ptr(weight))
        return weight


@dataclass
class KeyValueCacheEvictParam(KeyValueCacheParam):
    """Cache geometry, and the positions that stay whatever their weight: the first ``sink``, the last ``recent``."""
    sink: int = 0
    recent: int = 0


class KeyValueCacheEvict(_CacheOp):
    """Which cached positions to keep, per kv head: the last ``recent``, the first ``sink``, and the highest
    accumulated weights (ties: the lowest position) up to the sequence's budget.  Returns the kept positions
    [batch, num_kv_heads, max_budget] in ascending order, -1 behind them; KeyValueCacheCompact moves their rows."""

    def __init__(self, param: KeyValueCacheEvictParam):
        super().__init__(param)

    def forward(self, weight, cachestarts, kvlens, budgets, max_kvlen: int, max_budget: int,
                kept: torch.Tensor | None = None) -> torch.Tensor:
        a = self.param
        _require_cuda(weight=weight)
        if weight.dim() != 3:
            raise OpError("RC_INVALID_VALUE", "weight must be [num_layer, num_kv_heads, max_tokens]")
        device, heads, rows = weight.get_device(), weight.shape[1], weight.shape[2]
        self._check_weight(device, weight, heads, rows)
        _require(device, torch.int64, cachestarts=cachestarts, kvlens=kvlens, budgets=budgets)
        batch, max_budget = kvlens.numel(), int(max_budget)
        if kvlens.dim() != 1 or budgets.shape != kvlens.shape or max_budget < 0:
            raise OpError("RC_INVALID_VALUE", "budgets must have an entry per sequence and max_budget not be negative")
        if kept is None:
            kept = torch.empty((batch, heads, max_budget), dtype=torch.int64, device=weight.device)
        else:
            _require(device, torch.int64, kept=kept)
            if kept.shape != (batch, heads, max_budget):
                raise OpError("RC_INVALID_VALUE", "kept must be [batch, num_kv_heads, max_budget]")
        # the choice does not depend on the head size; any supported one describes the rows
        p = self._params(heads, heads, 128, batch, max_kvlen, rows, cachestarts)
        self._call("pplb200_kv_evict_select", self.lib.kv_evict_workspace_size, self.lib.kv_evict_select, p, device,
                   batch == 0 or max_budget == 0, _ptr(weight), _ptr(cachestarts), _ptr(kvlens), _ptr(budgets), a.sink, a.recent, max_budget, _ptr(kept))
        return kept


class KeyValueCacheCompact(_CacheOp):
    """Moves the cache rows of the kept positions to the front, in place: position base + kept[i] to base + i, of
    ``num_layers`` layers from layer_idx on.  ``kept`` [batch, num_kv_heads or 1, K] is strictly ascending and ends at
    its first negative entry, whatever follows it; ``kvlens`` are the positions the sequences had.  ``weight`` (as of AttentionWeight)
    moves along and is zeroed behind the kept positions."""

    def __init__(self, param: KeyValueCacheParam):
        super().__init__(param)

    def forward(self, kept, cachestarts, base, kvlens, max_kvlen: int, cache, scale, weight=None,
                num_layers: int = 1) -> None:
        device, heads, dim, rows = self._check_cache(cache, scale)
        _require(device, torch.int64, kept=kept, cachestarts=cachestarts, base=base, kvlens=kvlens)
        batch = kvlens.numel()
        if kvlens.dim() != 1 or kept.dim() != 3 or kept.shape[0] != batch or kept.shape[1] not in (1, heads) or base.shape != kvlens.shape:
            raise OpError("RC_INVALID_VALUE", "kept must be [batch, num_kv_heads or 1, K], base and kvlens [batch]")
        if weight is not None:
            self._check_weight(device, weight, heads, rows)
        p = self._params(heads, heads, dim, batch, max_kvlen, rows, cachestarts)
        _, kept_heads, most = kept.shape
        self._call("pplb200_kv_compact", lambda q: self.lib.kv_compact_workspace_size(q, kept_heads, most, num_layers),
                   self.lib.kv_compact, p, device, batch == 0 or (most == 0 and weight is None), _ptr(kept), kept_heads, most, _ptr(base), _ptr(kvlens),
                   _ptr(cachestarts), num_layers, _ptr(cache), _ptr(scale), _ptr(weight))
