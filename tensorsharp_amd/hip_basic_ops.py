"""Host-side operator facade of the HIP backend — the Python twin of a `HipBasicOps` class.

Names, argument meaning and error behaviour follow the quantized entry points of
TensorSharp.Backends.GGML/GgmlBasicOps.cs (:313-329 AddmmQuant, :689-704 AddmmQuantBatch,
:706-709 PreloadQuantizedWeight) and GgmlGgufTensorDequant.cs (:9-33 row size, :36-86 dequant).
ArgumentException -> ValueError, NotSupportedException -> NotImplementedError,
InvalidOperationException (native failure) -> RuntimeError.

Host tensors are numpy float32 arrays (the reference's tensors are host memory); device
tensors are torch CUDA tensors, which only supply memory and the stream.
"""
import ctypes as C

import numpy as np

from . import hip_native as N


class QuantizedWeight:
    """Raw GGUF blocks of one 2-D weight: twin of ModelBase.QuantizedWeight (TensorSharp.Models/ModelBase.cs:24-202).

    data        numpy uint8 array (host) or torch uint8 CUDA tensor (device) holding ne1 rows of row_size(type, ne0) bytes
    cache_key   the pointer the matmul entry points take as m2_data: the host address, or - after
                EnsureDeviceCacheKey() - an opaque key that stays valid once the host bytes are released
    An instance either owns its bytes (built from an array, or a concatenated copy) or is an external view of a larger
    buffer kept alive by `owner_token` (the GGUF mapping); adjacent external views of one owner concatenate without
    a copy."""

    def __init__(self, data, ggml_type, ne0, ne1, owner_token=None):
        self.ggml_type = int(ggml_type)
        self.ne0 = int(ne0)   # K, in features
        self.ne1 = int(ne1)   # N, out features
        self.data = data
        self.raw_bytes = int(data.numel() if hasattr(data, "numel") else data.size)
        self._owner_token = owner_token
        self._owns_buffer = owner_token is None
        self._key = None      # opaque device cache key (EnsureDeviceCacheKey)
        expect = HipBasicOps.GetRowSizeBytes(self.ggml_type, self.ne0) * self.ne1
        if self.raw_bytes < expect:
            raise ValueError(f"weight bytes {self.raw_bytes} < {expect} for {ne1}x{ne0} type {ggml_type}")

    # -- storage -----------------------------------------------------------------------------
    @property
    def is_device(self):
        return hasattr(self.data, "data_ptr")

    @property
    def HasHostData(self):
        return self.data is not None and not self.is_device

    @property
    def HasExternalHostView(self):
        return self.HasHostData and not self._owns_buffer and self._owner_token is not None

    @property
    def ptr(self):
        """what the matmul entry points receive: the cache key when the bytes were released, else the data address"""
        if self.data is None:
            if self._key is None:
                raise RuntimeError("Quantized weight has neither host data nor a device cache key.")
            return self._key
        return self.data.data_ptr() if self.is_device else self.data.ctypes.data

    @property
    def CacheKey(self):
        return self._key if self._key is not None else (0 if self.data is None else self.ptr)

    @staticmethod
    def AllocateBuffer(size):
        """64-byte aligned host bytes (ModelBase.cs:189-195)"""
        raw = np.empty(int(size) + 64, dtype=np.uint8)
        off = (-raw.ctypes.data) % 64
        return raw[off:off + int(size)]

    @staticmethod
    def CreateExternalView(data, ggml_type, ne0, ne1, owner_token):
        """A view of bytes owned by `owner_token` (ModelBase.cs:82-90)."""
        if data is None or (hasattr(data, "size") and data.size == 0):
            raise ValueError("External quantized weight view requires a non-empty data view.")
        if owner_token is None:
            raise ValueError("ownerToken must not be None.")
        return QuantizedWeight(data, ggml_type, ne0, ne1, owner_token=owner_token)

    @staticmethod
    def TryCreateConcatenatedView(*weights):
        """One weight of ne1 = sum(ne1) over byte-adjacent external views of the same owner, type and row length; None when
        the views do not qualify (ModelBase.cs:92-126)."""
        if len(weights) < 2 or weights[0] is None:
            return None
        first = weights[0]
        if not first.HasHostData or first._owns_buffer or first._owner_token is None:
            return None
        total_bytes = total_ne1 = 0
        expected = first.ptr
        for w in weights:
            if (w is None or not w.HasHostData or w._owns_buffer or w._owner_token is not first._owner_token or
                    w.ggml_type != first.ggml_type or w.ne0 != first.ne0 or w.ptr != expected):
                return None
            total_bytes += w.raw_bytes
            total_ne1 += w.ne1
            expected += w.raw_bytes
        span = (C.c_uint8 * total_bytes).from_address(first.ptr)
        data = np.frombuffer(span, dtype=np.uint8)
        fused = QuantizedWeight(data, first.ggml_type, first.ne0, total_ne1, owner_token=first._owner_token)
        fused._keepalive = [w.data for w in weights]     # the span borrows these views' memory
        return fused

    @staticmethod
    def ConcatOrCreateCopy(*weights):
        """Rows of the weights stacked in order: a view when they are adjacent in one mapping, else a copy into a fresh
        aligned buffer (ModelBase.cs:128-159)."""
        if len(weights) == 0 or weights[0] is None:
            raise ValueError("At least one quantized weight is required.")
        fused = QuantizedWeight.TryCreateConcatenatedView(*weights)
        if fused is not None:
            return fused
        first = weights[0]
        total = 0
        for w in weights:
            if w is None:
                raise ValueError("Quantized weight list cannot contain null entries.")
            if not w.HasHostData:
                raise RuntimeError("Cannot concatenate quantized weights after their host storage has been released.")
            total += w.raw_bytes
        buf = QuantizedWeight.AllocateBuffer(total)
        off = 0
        for w in weights:
            buf[off:off + w.raw_bytes] = w.data.reshape(-1)
            off += w.raw_bytes
        return QuantizedWeight(buf, first.ggml_type, first.ne0, sum(w.ne1 for w in weights))

    def EnsureDeviceCacheKey(self):
        """An opaque key for PreloadQuantizedWeight that outlives the host bytes (ModelBase.cs:161-170: a GCHandle there,
        the address of a small pinned-by-reference buffer here)."""
        if self._key is None:
            self._key_anchor = np.zeros(1, dtype=np.uint8)
            self._key = self._key_anchor.ctypes.data
        return self._key

    def ReleaseHostData(self):
        """Drop the host bytes (ModelBase.cs:172-187); the weight stays usable through its device cache key."""
        self.data = None
        self._owns_buffer = False
        self._owner_token = None
        self._keepalive = None

    def Dispose(self):
        self.ReleaseHostData()
        self._key = None


def FuseGateUpWeights(quant_weights, num_layers):
    """Twin of ModelBase.FuseGateUpWeights (ModelBase.cs:768-802) for the quantized branch: blk.L.ffn_gate.weight and
    blk.L.ffn_up.weight of equal type and row length become blk.L.ffn_gate_up.weight (gate rows, then up rows); the two
    originals are removed and disposed.  Returns the number of layers fused."""
    fused = 0
    for layer in range(int(num_layers)):
        gate_name, up_name = f"blk.{layer}.ffn_gate.weight", f"blk.{layer}.ffn_up.weight"
        gw, uw = quant_weights.get(gate_name), quant_weights.get(up_name)
        if gw is None or uw is None or gw.ggml_type != uw.ggml_type or gw.ne0 != uw.ne0:
            continue
        quant_weights[f"blk.{layer}.ffn_gate_up.weight"] = QuantizedWeight.ConcatOrCreateCopy(gw, uw)
        del quant_weights[gate_name], quant_weights[up_name]
        gw.Dispose()
        uw.Dispose()
        fused += 1
    return fused


def FuseExpertGateUpWeights(quant_weights, num_layers, num_experts, biases=None):
    """Twin of GptOssModel.FuseExpertGateUpWeights (GptOssModel.cs:126-180): per layer and expert,
    blk.L.ffn_gate_exps.E.weight and blk.L.ffn_up_exps.E.weight of equal type and row length become
    blk.L.ffn_gate_up_exps.E.weight (gate rows, then up rows; a copy, since gate and up live in different tensors of the
    file).  `biases` (name -> float32 array [1, n], the split biases of GptOssModel.cs:95-121) are fused the same way.
    Returns the number of experts fused."""
    fused = 0
    for layer in range(int(num_layers)):
        for e in range(int(num_experts)):
            gate_name, up_name = f"blk.{layer}.ffn_gate_exps.{e}.weight", f"blk.{layer}.ffn_up_exps.{e}.weight"
            gw, uw = quant_weights.get(gate_name), quant_weights.get(up_name)
            if gw is not None and uw is not None and gw.ggml_type == uw.ggml_type and gw.ne0 == uw.ne0:
                quant_weights[f"blk.{layer}.ffn_gate_up_exps.{e}.weight"] = QuantizedWeight.ConcatOrCreateCopy(gw, uw)
                del quant_weights[gate_name], quant_weights[up_name]
                gw.Dispose()
                uw.Dispose()
                fused += 1
            if biases is not None:
                gb_name, ub_name = f"blk.{layer}.ffn_gate_exps.{e}.bias", f"blk.{layer}.ffn_up_exps.{e}.bias"
                if gb_name in biases and ub_name in biases:
                    biases[f"blk.{layer}.ffn_gate_up_exps.{e}.bias"] = np.concatenate(
                        [biases.pop(gb_name).reshape(1, -1), biases.pop(ub_name).reshape(1, -1)], axis=1)
    return fused


def SplitExpertBiases(float_weights, num_layers):
    """Twin of GptOssModel.SplitExpertBiases (GptOssModel.cs:93-124): blk.L.ffn_{gate,up,down}_exps.bias [E, n] become
    blk.L.ffn_*_exps.E.bias [1, n].  Returns the number of tensors split."""
    split = 0
    for layer in range(int(num_layers)):
        for kind in ("ffn_gate_exps", "ffn_up_exps", "ffn_down_exps"):
            name = f"blk.{layer}.{kind}.bias"
            if name not in float_weights:
                continue
            b = float_weights.pop(name)
            for e in range(b.shape[0]):
                float_weights[f"blk.{layer}.{kind}.{e}.bias"] = np.ascontiguousarray(b[e]).reshape(1, -1)
            split += 1
    return split


def StackExpertWeights(weights):
    """One weight holding the rows of all experts in order ([E * ne1] rows), the operand of
    HipBasicOps.MoEExpertsGptOssForward: a view when the experts are byte-adjacent views of one mapping (a `*_exps.` tensor
    split by GgufFile.expert_weights), else a copy into one aligned buffer (experts fused from two tensors)."""
    if len(weights) == 1:
        return weights[0]
    return QuantizedWeight.ConcatOrCreateCopy(*weights)


def FuseQKVWeights(quant_weights, num_layers):
    """Twin of the models' FuseQKVWeights (Qwen3Model.cs:57-85): attn_q / attn_k / attn_v of equal type and row length
    become blk.L.attn_qkv.weight."""
    fused = 0
    for layer in range(int(num_layers)):
        names = [f"blk.{layer}.attn_{p}.weight" for p in "qkv"]
        ws = [quant_weights.get(n) for n in names]
        if any(w is None for w in ws) or any(w.ggml_type != ws[0].ggml_type or w.ne0 != ws[0].ne0 for w in ws):
            continue
        quant_weights[f"blk.{layer}.attn_qkv.weight"] = QuantizedWeight.ConcatOrCreateCopy(*ws)
        for n, w in zip(names, ws):
            del quant_weights[n]
            w.Dispose()
        fused += 1
    return fused


def _host_view(a, standard):
    if not isinstance(a, np.ndarray) or a.ndim != 2:
        raise ValueError("AddmmQuant requires 2D tensors for result and m1.")
    if a.dtype != np.float32:
        raise ValueError("AddmmQuant requires Float32 tensors for result and m1.")
    s0, s1 = a.strides[0] // 4, a.strides[1] // 4
    if a.strides[0] % 4 or a.strides[1] % 4 or s0 < 0 or s1 < 0 or (standard and s1 != 1):
        raise NotImplementedError("HIP AddmmQuant requires tensors with supported row-contiguous layouts.")
    span = ((a.shape[0] - 1) * s0 + (a.shape[1] - 1) * s1 + 1) * 4
    return N.TensorView2D(a.ctypes.data, a.shape[0], a.shape[1], s0, s1, span)


_torch_module = None


def _torch():
    """torch, imported with the first call that meets device tensors.  The host path of a call is written for its length: a
    GEMV of one token takes 8 us on the device, and an import statement, a stream object or a shape read three times over
    cost up to a microsecond each (one Q8_0 9728 x 2560 linear after another: 12.7 -> 9.1 us of host time per call)."""
    global _torch_module
    if _torch_module is None:
        import torch
        _torch_module = torch
    return _torch_module


def _device_view(t):
    torch = _torch()
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise ValueError("AddmmQuant requires 2D tensors for result and m1.")
    if t.dtype != torch.float32:
        raise ValueError("AddmmQuant requires Float32 tensors for result and m1.")
    if not t.is_cuda:
        raise ValueError("device AddmmQuant requires tensors in GPU memory.")
    rows, cols = t.shape
    s0, s1 = t.stride()
    if s1 != 1 and cols > 1:
        raise NotImplementedError("HIP AddmmQuant requires tensors with supported row-contiguous layouts.")
    return N.TensorView2D(t.data_ptr(), rows, cols, s0, 1, ((rows - 1) * s0 + cols) * 4)


def _vector(t, dtype, count, name, device):
    """address of a contiguous vector of `count` values on that device (its index); None stays None"""
    if t is None:
        return None
    if t.dtype is not dtype or t.numel() != count or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {str(dtype).split('.')[-1]} tensor of {count} values.")
    if t.get_device() != device:
        raise ValueError(f"{name} is not on the device of the other tensors.")
    return t.data_ptr()


def _use_stream_of(device):
    """Launches go to the current stream, which is one of the current device: tensors of another one have no stream here."""
    torch = _torch()
    try:                                        # (see UseCurrentStream)
        current = torch._C._cuda_getDevice()
        handle = torch._C._cuda_getCurrentRawStream(current)
    except AttributeError:
        current = torch.cuda.current_device()
        handle = torch.cuda.current_stream().cuda_stream
    if device != current:
        raise ValueError("the tensors must be on the current device.")
    N.lib().TSHip_SetStream(handle)


def _device_view3(t, name):
    torch = _torch()
    if t.dim() != 3 or t.dtype is not torch.float32:
        raise ValueError(f"{name} requires 3D Float32 tensors.")
    if not t.is_cuda:
        raise ValueError(f"{name} requires tensors in GPU memory of one device.")
    d0, d1, d2 = t.shape
    s0, s1, s2 = t.stride()
    return N.TensorView3D(t.data_ptr(), d0, d1, d2, s0, s1, s2, ((d0 - 1) * s0 + (d1 - 1) * s1 + (d2 - 1) * s2 + 1) * 4)


class RotaryPositions:
    """How positions turn a head (the descriptor of RoPE and RoPEStorePaged): the first `dims` dimensions in adjacent pairs (mode 0) or
    in halves (mode 2), pair i by position * base^(-2 i / dims) radians.  freq_factors (float32 device tensor [dims / 2]) divide the
    frequencies, freq_scale multiplies them (a context n times as long: 1 / n); with ext_factor above 0 only those of pairs that turn
    less than beta_slow times over original_context, those between beta_slow and beta_fast in part, and the result is
    multiplied by 1 + 0.1 ln(1 / freq_scale).  attn_factor multiplies it too."""

    def __init__(self, dims, mode=2, base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0,
                 original_context=0, freq_factors=None):
        address = None
        self.device = None                       # of freq_factors; without them any
        if freq_factors is not None:
            torch = _torch()
            if not freq_factors.is_cuda:
                raise ValueError("freq_factors must be in GPU memory.")
            self.device = freq_factors.get_device()
            address = _vector(freq_factors, torch.float32, int(dims) // 2, "freq_factors", self.device)
        self._keepalive = freq_factors
        self.native = N.Rope(int(dims), int(mode), float(base), float(freq_scale), float(ext_factor), float(attn_factor), float(beta_fast),
                             float(beta_slow), int(original_context), address)
        self.ref = C.byref(self.native)

    def _elsewhere(self):
        raise ValueError("freq_factors is not on the device of the other tensors.")


class PagedKVCache:
    """Keys and values of many sequences in pages: k and v [pages, tokens of a page, kv heads, head_dim] device tensors of float32, float16 or
    bfloat16 (any strides with contiguous rows of head_dim, so that heads may lie before tokens in memory), page_table [sequences,
    pages of a sequence] int32 on the device.  Position p of sequence s is token p % page_size of page page_table[s, p // page_size]; an
    entry outside the pages stands for none.  The contiguous cache [kv heads, max_seq, head_dim] of the whole-layer
    decode is one page: PagedKVCache(k.transpose(0, 1)[None], v.transpose(0, 1)[None], table of one 0).

    In four bits (MXFP4: blocks of 32 along a head): k and v uint8 [pages, tokens, kv heads, head_dim / 2], two codes a byte with the first
    dimension's in the lower bits, k_scales and v_scales uint8 [pages, tokens, kv heads, head_dim / 32].  A code is sign, two bits of exponent and
    one of mantissa (0, 0.5, 1, 1.5, 2, 3, 4, 6) and stands for that times 2^(scale - 127), for NaN where the scale is 255."""

    def __init__(self, k, v, page_table, k_scales=None, v_scales=None):
        torch = _torch()
        types = {torch.float32: N.TYPE_F32, torch.float16: N.TYPE_F16, torch.bfloat16: N.TYPE_BF16, torch.uint8: N.TYPE_MXFP4}
        if k.dim() != 4 or k.shape != v.shape:
            raise ValueError("PagedKVCache requires 4D tensors of one shape for k and v.")
        if k.dtype not in types or v.dtype != k.dtype:
            raise ValueError("PagedKVCache requires Float32, Float16 or BFloat16 keys and values of one type, or UInt8 codes.")
        four, head_dim, scales = k.dtype is torch.uint8, k.shape[3], ()
        if four != (k_scales is not None) or four != (v_scales is not None):
            raise ValueError("PagedKVCache requires k_scales and v_scales with codes of four bits, and only with those.")
        if four:
            head_dim *= 2
            if k_scales.dtype is not torch.uint8 or v_scales.dtype is not torch.uint8 or head_dim % 32 != 0 or \
                    tuple(k_scales.shape) != (*k.shape[:3], head_dim // 32) or v_scales.shape != k_scales.shape:
                raise ValueError("PagedKVCache requires UInt8 scales [pages, tokens, kv heads, head_dim / 32], head_dim a multiple of 32.")
            if k_scales.device != k.device or v_scales.device != k.device:
                raise ValueError("PagedKVCache requires tensors in GPU memory of one device.")
            if head_dim > 32 and (k_scales.stride(3) != 1 or v_scales.stride(3) != 1):
                raise NotImplementedError("PagedKVCache requires contiguous rows of scales.")
            scales = (k_scales.data_ptr(), v_scales.data_ptr(), *k_scales.stride()[:3], *v_scales.stride()[:3])
        if page_table.dim() != 2 or page_table.dtype != torch.int32:
            raise ValueError("PagedKVCache requires a 2D Int32 page table.")
        if max(*k.shape[1:3], *page_table.shape) >= 2 ** 31:          # (the call takes 32 bits of them)
            raise ValueError("PagedKVCache requires fewer than 2^31 tokens of a page, heads, sequences and pages of a sequence.")
        if not k.is_cuda or v.device != k.device or page_table.device != k.device:
            raise ValueError("PagedKVCache requires tensors in GPU memory of one device.")
        if k.stride(3) != 1 or v.stride(3) != 1 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
            raise NotImplementedError("PagedKVCache requires contiguous rows of head_dim and of the page table.")
        self.k, self.v, self.page_table, self.k_scales, self.v_scales = k, v, page_table, k_scales, v_scales
        self.num_kv_heads, self.head_dim, self.num_seqs = k.shape[2], head_dim, page_table.shape[0]
        self.native = N.PagedCache(k.data_ptr(), v.data_ptr(), types[k.dtype], k.shape[2], head_dim, k.shape[1], k.shape[0], *k.stride()[:3],
                                   *v.stride()[:3], page_table.data_ptr(), page_table.stride(0), page_table.shape[0], page_table.shape[1], *scales)
        self.ref = C.byref(self.native)
        self.device = k.get_device()

    def _sequences(self, row_starts, context_lens, i32):
        return (_vector(row_starts, i32, self.num_seqs + 1, "row_starts", self.device),
                _vector(context_lens, i32, self.num_seqs, "context_lens", self.device))


class PagePool:
    """Pages that sequences share, for the caches of all layers: page_table [sequences, pages of a sequence] int32 (the one of the PagedKVCaches),
    references [pages] int32 (how many sequences have a page, 0: free), context_lens [sequences] int32 (tokens), all on one device and changed in place by
    ResizeSequences, ForkSequences and CompactPages.  A sequence has the pages of its first ceil(tokens / page_size) entries, behind them is -1: an empty
    pool is a table of -1 and zeros.  It keeps scratch of its own (an int32 for each entry of the table and for each page): keep the pool until the work of its calls,
    and graphs that have captured them, are done with."""

    def __init__(self, page_table, references, context_lens, page_size):
        torch = _torch()
        if not 0 < page_size < 2 ** 31 or any(n >= 2 ** 31 for n in page_table.shape):          # (the calls take 32 bits of them)
            raise ValueError("PagePool requires a page size of 1 to 2^31 - 1 tokens, and fewer than 2^31 sequences and pages of a sequence.")
        if page_table.dim() != 2 or page_table.dtype != torch.int32 or not page_table.is_cuda:
            raise ValueError("PagePool requires a 2D Int32 page table in GPU memory.")
        if page_table.shape[1] > 1 and page_table.stride(1) != 1:
            raise NotImplementedError("PagePool requires contiguous rows of the page table.")
        self.device = page_table.get_device()
        self.num_seqs, self.num_pages = page_table.shape[0], references.numel()
        addresses = (_vector(references, torch.int32, self.num_pages, "references", self.device),
                     _vector(context_lens, torch.int32, self.num_seqs, "context_lens", self.device))
        count = N.lib().TSHip_PagePoolScratchDevice(self.num_seqs, page_table.shape[1], self.num_pages)
        if count == 0:
            raise ValueError("PagePool requires 1 to 65535 sequences and 1 to 2^28 pages.")
        self.page_table, self.references, self.context_lens, self.page_size = page_table, references, context_lens, int(page_size)
        self._scratch = torch.empty((count,), dtype=torch.int32, device=page_table.device)
        self.native = N.PagePool(page_table.data_ptr(), page_table.stride(0), self.num_seqs, page_table.shape[1], self.page_size, self.num_pages, *addresses,
                                 self._scratch.data_ptr())
        self.ref = C.byref(self.native)

    def _moves(self, moves, count):
        """address of a list of pairs, `count` of them (None: as many as there are)"""
        return _pairs(moves, count, self.device)


def _pairs(moves, count, device):
    if moves is None or moves.dim() != 2 or moves.shape[1] != 2 or (count is not None and moves.shape[0] != count):
        raise ValueError(f"moves must be an Int32 tensor [{count if count is not None else 'moves'}, 2].")
    if moves.shape[0] >= 2 ** 31:                    # (the calls take 32 bits of it)
        raise ValueError("moves must be fewer than 2^31 pairs.")
    return _vector(moves, _torch().int32, moves.shape[0] * 2, "moves", device)


class HipBasicOps:
    """Static quantized-matmul entry points of the HIP backend."""

    @staticmethod
    def IsAvailable():
        return N.lib().TSHip_IsBackendAvailable(N.BACKEND_HIP) == 1

    @staticmethod
    def GetRowSizeBytes(ggml_type, ne0):
        rb = N.lib().TSHip_RowSize(int(ggml_type), int(ne0))
        if rb <= 0:
            raise NotImplementedError(
                f"GGML tensor type {ggml_type} is not supported, or ne[0]={ne0} is not aligned to the type block size.")
        return int(rb)

    # -- dequantization -------------------------------------------------------------------
    @staticmethod
    def DequantizeToFloat32(ggml_type, src, num_elements):
        """Host bytes -> host fp32 (computed on the GPU).  Codes as GgmlNative.cs:1493-1503."""
        if not isinstance(src, np.ndarray) or src.dtype != np.uint8:
            raise ValueError("Source must be a uint8 array.")
        if num_elements < 0:
            raise ValueError("numElements out of range.")
        dst = np.empty(int(num_elements), dtype=np.float32)
        rc = N.lib().TSHip_DequantizeToF32(int(ggml_type), src.ctypes.data, int(num_elements), dst.ctypes.data)
        if rc == -2:
            raise NotImplementedError(f"HIP backend cannot dequantize GGUF tensor type {ggml_type}.")
        if rc != 0:
            raise RuntimeError(f"Native HIP dequantization failed (code {rc}): {N.get_last_error()}")
        return dst

    @staticmethod
    def DequantizeToFloat32Device(ggml_type, src, num_elements, dst=None):
        import torch
        if dst is None:
            dst = torch.empty(int(num_elements), dtype=torch.float32, device=src.device)
        HipBasicOps.UseCurrentStream()
        rc = N.lib().TSHip_DequantizeToF32Device(int(ggml_type), src.data_ptr(), int(num_elements), dst.data_ptr())
        if rc == -2:
            raise NotImplementedError(f"HIP backend cannot dequantize GGUF tensor type {ggml_type}.")
        if rc != 0:
            raise RuntimeError(f"Native HIP dequantization failed (code {rc}): {N.get_last_error()}")
        return dst

    # -- fused wrappers (GgmlBasicOps.FusedRmsNormMatMulQuant / FusedMatMulQuantAdd / FusedFFNSwiGLUQuant) ------
    @staticmethod
    def _views(out, inp):
        """host (numpy) or device (torch) views of the in/out pair and the export suffix that takes them"""
        if isinstance(out, np.ndarray):
            return _host_view(out, standard=True), _host_view(inp, standard=False), ""
        return _device_view(out), _device_view(inp), "Device"

    @staticmethod
    def _addr(a):
        return a.ctypes.data if isinstance(a, np.ndarray) else a.data_ptr()

    @staticmethod
    def FusedRmsNormMatMulQuant(result, input, norm_weight, eps, weight):
        """result = (RMSNorm(input) * norm_weight) * W^T; all host (numpy) or all device (torch) tensors."""
        rv, iv, sfx = HipBasicOps._views(result, input)
        fn = getattr(N.lib(), "TSHip_FusedRmsNormMatMulQuantF32" + sfx)
        ok = fn(rv, iv, C.c_void_p(HipBasicOps._addr(norm_weight)), int(norm_weight.shape[0]), float(eps),
                C.c_void_p(weight.ptr), weight.ggml_type, weight.ne0, weight.ne1, weight.raw_bytes)
        N.check_result(ok, "fused_rms_norm_matmul_quant")

    @staticmethod
    def FusedMatMulQuantAdd(residual, input, weight):
        """residual += input * W^T, in place."""
        rv, iv, sfx = HipBasicOps._views(residual, input)
        fn = getattr(N.lib(), "TSHip_FusedMatMulQuantAddF32" + sfx)
        ok = fn(rv, iv, C.c_void_p(weight.ptr), weight.ggml_type, weight.ne0, weight.ne1, weight.raw_bytes)
        N.check_result(ok, "fused_matmul_quant_add")

    @staticmethod
    def FusedFFNSwiGLUQuant(residual, input, norm_weight, eps, gate_up, down, half_dim):
        """residual += W_down * (silu(g) * u), [g | u] = W_gate_up * (RMSNorm(input) * norm_weight)."""
        rv, iv, sfx = HipBasicOps._views(residual, input)
        fn = getattr(N.lib(), "TSHip_FusedFFNSwiGLUQuantF32" + sfx)
        ok = fn(rv, iv, C.c_void_p(HipBasicOps._addr(norm_weight)), int(norm_weight.shape[0]), float(eps),
                C.c_void_p(gate_up.ptr), gate_up.ggml_type, gate_up.ne0, gate_up.ne1, gate_up.raw_bytes,
                C.c_void_p(down.ptr), down.ggml_type, down.ne0, down.ne1, down.raw_bytes, int(half_dim))
        N.check_result(ok, "fused_ffn_swiglu_quant")

    @staticmethod
    def _weight_args(w):
        return (C.c_void_p(w.ptr), w.ggml_type, w.ne0, w.ne1, w.raw_bytes)

    @staticmethod
    def FusedOutProjFFN(residual, input, out_proj, ffn_norm_weight, eps, gate_up, down, half_dim):
        """residual += input * W_out^T, then residual += W_down * (silu(g) * u) with [g | u] = W_gate_up * (RMSNorm(residual) *
        ffn_norm_weight) (GgmlBasicOps.cs:449-480).  All host (numpy) or all device (torch) tensors."""
        rv, iv, sfx = HipBasicOps._views(residual, input)
        fn = getattr(N.lib(), "TSHip_FusedOutProjFFNQuantF32" + sfx)
        ok = fn(rv, iv, *HipBasicOps._weight_args(out_proj), C.c_void_p(HipBasicOps._addr(ffn_norm_weight)),
                int(ffn_norm_weight.shape[0]), float(eps), *HipBasicOps._weight_args(gate_up), *HipBasicOps._weight_args(down),
                int(half_dim))
        N.check_result(ok, "fused_outproj_ffn")

    @staticmethod
    def FusedOutProjNormRouter(residual, input, out_proj, norm_weight, eps, normed_output, router, router_output):
        """residual += input * W_out^T; normed_output = RMSNorm(residual) * norm_weight; router_output = normed_output *
        W_router^T (GgmlBasicOps.cs:416-447).  The router weight may be F32 / F16 / BF16 or a block format."""
        rv, iv, sfx = HipBasicOps._views(residual, input)
        view = (lambda a: _host_view(a, standard=True)) if sfx == "" else _device_view
        fn = getattr(N.lib(), "TSHip_FusedOutProjNormRouterQuantF32" + sfx)
        ok = fn(rv, iv, *HipBasicOps._weight_args(out_proj), C.c_void_p(HipBasicOps._addr(norm_weight)),
                int(norm_weight.shape[0]), float(eps), view(normed_output), *HipBasicOps._weight_args(router),
                view(router_output))
        N.check_result(ok, "fused_outproj_norm_router")

    @staticmethod
    def _expert_ptrs(weights):
        return (C.c_void_p * len(weights))(*[w.ptr for w in weights])

    @staticmethod
    def _shape_args(w):
        return (w.ggml_type, w.ne0, w.ne1, w.raw_bytes)

    @staticmethod
    def MoEExpertsForward(result, input, up, down, route_weights):
        """result = sum_e route_weights[e] * W_down[e] * relu(W_up[e] * input)^2 for up to 16 selected experts
        (GgmlBasicOps.cs:586-613; Nemotron).  up / down: lists of QuantizedWeight sharing type and shape."""
        rv, iv, sfx = HipBasicOps._views(result, input)
        n = len(up)
        rw = (C.c_float * n)(*[float(v) for v in route_weights])
        fn = getattr(N.lib(), "TSHip_MoEExpertsForwardF32" + sfx)
        ok = fn(rv, iv, n, HipBasicOps._expert_ptrs(up), HipBasicOps._expert_ptrs(down), *HipBasicOps._shape_args(up[0]),
                *HipBasicOps._shape_args(down[0]), rw)
        N.check_result(ok, "moe_experts_forward")

    @staticmethod
    def MoEExpertsSwiGLUForward(result, input, gate, up, down, route_weights):
        """result = sum_e route_weights[e] * W_down[e] * (silu(W_gate[e] x) * (W_up[e] x)) (GgmlBasicOps.cs:615-645)."""
        rv, iv, sfx = HipBasicOps._views(result, input)
        n = len(up)
        rw = (C.c_float * n)(*[float(v) for v in route_weights])
        fn = getattr(N.lib(), "TSHip_MoEExpertsSwiGLUForwardF32" + sfx)
        ok = fn(rv, iv, n, HipBasicOps._expert_ptrs(gate), HipBasicOps._expert_ptrs(up), HipBasicOps._expert_ptrs(down),
                *HipBasicOps._shape_args(gate[0]), *HipBasicOps._shape_args(up[0]), *HipBasicOps._shape_args(down[0]), rw)
        N.check_result(ok, "moe_experts_swiglu_forward")

    @staticmethod
    def MoEExpertsSwiGLUResidual(residual, input, gate, up, down, route_weights, shared=None, shared_scalar=1.0):
        """residual += sum_e route_weights[e] * expert_e(input) [+ shared_scalar * shared_expert(input)]
        (GgmlBasicOps.cs:647-700); shared = (gate, up, down) QuantizedWeights or None; up to 32 routed experts."""
        rv, iv, sfx = HipBasicOps._views(residual, input)
        n = len(up)
        rw = (C.c_float * n)(*[float(v) for v in route_weights])
        if shared is None:
            sh = (0, None, None, None, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
        else:
            sh = (1, C.c_void_p(shared[0].ptr), C.c_void_p(shared[1].ptr), C.c_void_p(shared[2].ptr),
                  *HipBasicOps._shape_args(shared[0]), *HipBasicOps._shape_args(shared[1]), *HipBasicOps._shape_args(shared[2]))
        fn = getattr(N.lib(), "TSHip_MoEExpertsSwiGLUResidualF32" + sfx)
        ok = fn(rv, iv, n, HipBasicOps._expert_ptrs(gate), HipBasicOps._expert_ptrs(up), HipBasicOps._expert_ptrs(down),
                *HipBasicOps._shape_args(gate[0]), *HipBasicOps._shape_args(up[0]), *HipBasicOps._shape_args(down[0]), rw,
                *sh, float(shared_scalar))
        N.check_result(ok, "moe_experts_swiglu_residual")

    @staticmethod
    def _view3(a):
        """3-D fp32 view of a numpy array or a torch CUDA tensor (strides in elements)"""
        host = isinstance(a, np.ndarray)
        if (a.ndim if host else a.dim()) != 3 or str(a.dtype).split(".")[-1] != "float32":
            raise ValueError("MulMatId requires 3D Float32 tensors.")
        st = [v // 4 for v in a.strides] if host else list(a.stride())
        span = (sum((d - 1) * s for d, s in zip(a.shape, st)) + 1) * 4
        return N.TensorView3D(HipBasicOps._addr(a), a.shape[0], a.shape[1], a.shape[2], st[0], st[1], st[2], span)

    @staticmethod
    def MulMatId(result, expert_weights, input, ids):
        """result[t, s, :] = expert_weights[ids[t, s]] @ input[t, s % slots] with F32 experts [E, rows, K]
        (GgmlNative.MulMatId, GgmlNative.cs:1076-1079).  All host (numpy; ids int32 or float32) or all device (torch; ids
        int32) tensors."""
        host = isinstance(result, np.ndarray)
        rows, cols = int(ids.shape[0]), int(ids.shape[1])
        if host:
            idc = np.ascontiguousarray(ids)
            if idc.dtype not in (np.int32, np.float32):
                raise ValueError("MulMatId ids must be Int32 or Float32.")
            desc = N.ContiguousTensor(idc.ctypes.data, int(idc.size), 3 if idc.dtype == np.int32 else 0)
            ok = N.lib().TSHip_MulMatIdF32(HipBasicOps._view3(result), HipBasicOps._view3(expert_weights),
                                           HipBasicOps._view3(input), desc, rows, cols)
        else:
            HipBasicOps.UseCurrentStream()
            ok = N.lib().TSHip_MulMatIdF32Device(HipBasicOps._view3(result), HipBasicOps._view3(expert_weights),
                                                 HipBasicOps._view3(input), C.c_void_p(ids.contiguous().data_ptr()), rows, cols)
        N.check_result(ok, "mulmatid")

    @staticmethod
    def AddId(result, src, bias, ids):
        """result[t, s, :] = src[t, s, :] + bias[ids[t, s], :] (GgmlBasicOps.AddID, GgmlBasicOps.cs:1092-1108; the bias of
        a MulMatId).  All host (numpy; ids int32 or float32) or all device (torch; ids int32) tensors; result may be src."""
        host = isinstance(result, np.ndarray)
        if (ids.ndim if host else ids.dim()) != 2 or (bias.ndim if host else bias.dim()) != 2:
            raise NotImplementedError("addid expects 2D bias and id tensors.")
        rows, cols = int(ids.shape[0]), int(ids.shape[1])
        if host:
            idc = np.ascontiguousarray(ids)
            if idc.dtype not in (np.int32, np.float32):
                raise ValueError("AddId ids must be Int32 or Float32.")
            desc = N.ContiguousTensor(idc.ctypes.data, int(idc.size), 3 if idc.dtype == np.int32 else 0)
            ok = N.lib().TSHip_AddIdF32(HipBasicOps._view3(result), HipBasicOps._view3(src), _host_view(bias, standard=True), desc, rows, cols)
        else:
            HipBasicOps.UseCurrentStream()
            ok = N.lib().TSHip_AddIdF32Device(HipBasicOps._view3(result), HipBasicOps._view3(src), _device_view(bias),
                                              C.c_void_p(ids.contiguous().data_ptr()), rows, cols)
        N.check_result(ok, "addid")

    # -- embedding gather ------------------------------------------------------------------
    @staticmethod
    def GetRowsQuant(result, weight_data, ggml_type, ne0, ne1, raw_bytes, indices):
        """result[i] = dequantized row indices[i] (GgmlBasicOps.cs:565-579). Host tensors; weight_data: address."""
        if not isinstance(result, np.ndarray) or result.ndim != 2 or result.dtype != np.float32:
            raise ValueError("GetRowsQuant requires a 2D Float32 result tensor.")
        idx = np.asarray(indices)
        if idx.dtype != np.int32 or not idx.flags["C_CONTIGUOUS"]:
            raise NotImplementedError("HIP GetRowsQuant requires a standard-layout result and contiguous Int32 indices.")
        rv = _host_view(result, standard=True)
        desc = N.ContiguousTensor(idx.ctypes.data, int(idx.size), 3)
        ok = N.lib().TSHip_GetRowsQuantF32(rv, C.c_void_p(weight_data), int(ggml_type), int(ne0), int(ne1),
                                           int(raw_bytes), desc)
        N.check_result(ok, "get_rows_quant")

    @staticmethod
    def GetRowsQuantDevice(result, weight, indices):
        """Device form: result [n x K] fp32 CUDA tensor, weight a device QuantizedWeight, indices int32 CUDA tensor."""
        rv = _device_view(result)
        ok = N.lib().TSHip_GetRowsQuantF32Device(rv, C.c_void_p(weight.ptr), weight.ggml_type, weight.ne0, weight.ne1,
                                                 weight.raw_bytes, C.c_void_p(indices.data_ptr()), int(indices.numel()))
        N.check_result(ok, "get_rows_quant")

    # -- matmul ---------------------------------------------------------------------------
    @staticmethod
    def AddmmQuant(result, m1, weight_data, ggml_type, ne0, ne1, raw_bytes):
        """result = m1 * W^T with host tensors (GgmlBasicOps.cs:313-329). weight_data: address (int)."""
        rv = _host_view(result, standard=True)
        mv = _host_view(m1, standard=False)
        ok = N.lib().TSHip_AddmmQuantF32(rv, mv, C.c_void_p(weight_data), int(ggml_type), int(ne0), int(ne1),
                                         int(raw_bytes))
        N.check_result(ok, "addmm_quant")

    @staticmethod
    def AddmmQuantDevice(result, m1, weight_data, ggml_type, ne0, ne1, raw_bytes):
        """Same contract with every pointer in device memory; asynchronous on the current stream."""
        rv = _device_view(result)
        mv = _device_view(m1)
        # (c_void_p refuses bytes, strings and arrays, which the bare argument would pass as host memory)
        ok = N.lib().TSHip_AddmmQuantF32Device(rv, mv, C.c_void_p(weight_data), int(ggml_type), int(ne0), int(ne1),
                                               int(raw_bytes))
        N.check_result(ok, "addmm_quant")

    @staticmethod
    def AddmmQuantDeviceNoAlloc(result, m1, weight_data, ggml_type, ne0, ne1, raw_bytes):
        """AddmmQuantDevice for callers that cannot allocate device memory: scratch lives in a static device array."""
        rv = _device_view(result)
        mv = _device_view(m1)
        ok = N.lib().TSHip_AddmmQuantF32DeviceNoAlloc(rv, mv, C.c_void_p(weight_data), int(ggml_type), int(ne0), int(ne1),
                                                      int(raw_bytes))
        N.check_result(ok, "addmm_quant")

    @staticmethod
    def PrepareGroup(results, m1s, weights):
        """Marshal a list of (result, m1, QuantizedWeight) problems once; returns the argument pack
        that AddmmQuantGroupDevice launches (decode loops reuse the pack every token)."""
        n = len(weights)
        if not (n == len(results) == len(m1s)) or n == 0:
            raise ValueError("results, m1s and weights must be equally long and non-empty.")
        t = weights[0].ggml_type
        if any(w.ggml_type != t for w in weights):
            raise ValueError("all weights of a group must share one block type.")
        rv = (N.TensorView2D * n)(*[_device_view(r) for r in results])
        mv = (N.TensorView2D * n)(*[_device_view(m) for m in m1s])
        wp = (C.c_void_p * n)(*[w.ptr for w in weights])
        ne0 = (C.c_int64 * n)(*[w.ne0 for w in weights])
        ne1 = (C.c_int64 * n)(*[w.ne1 for w in weights])
        rb = (C.c_int64 * n)(*[w.raw_bytes for w in weights])
        return (n, rv, mv, wp, t, ne0, ne1, rb)

    @staticmethod
    def AddmmQuantGroupDevice(pack):
        """count independent AddmmQuantDevice problems; one launch when all are decode GEMVs."""
        ok = N.lib().TSHip_AddmmQuantGroupF32Device(*pack)
        N.check_result(ok, "addmm_quant_group")

    @staticmethod
    def AddmmQuantBatch(result, m1, weight_data, ggml_type, ne0, raw_bytes, weight_offsets, weight_ne1):
        """Row b of m1 times the sub-weight at weight_offsets[b] (GgmlBasicOps.cs:689-704)."""
        rv = _host_view(result, standard=True)
        mv = _host_view(m1, standard=False)
        n = len(weight_offsets)
        if n != len(weight_ne1):
            raise ValueError("weight_offsets and weight_ne1 must have the same length.")
        offs = (C.c_int64 * n)(*[int(v) for v in weight_offsets])
        ne1s = (C.c_int64 * n)(*[int(v) for v in weight_ne1])
        ok = N.lib().TSHip_AddmmQuantBatchF32(rv, mv, C.c_void_p(weight_data), int(ggml_type), int(ne0),
                                              int(raw_bytes), n, offs, ne1s)
        N.check_result(ok, "addmm_quant_batch")

    @staticmethod
    def PreloadQuantizedWeight(cache_key, host_data, ggml_type, ne0, ne1, raw_bytes):
        ok = N.lib().TSHip_PreloadQuantizedWeight(C.c_void_p(cache_key), C.c_void_p(host_data), int(ggml_type),
                                                  int(ne0), int(ne1), int(raw_bytes))
        N.check_result(ok, "preload_quantized_weight")

    @staticmethod
    def InvalidateHostBuffer(ptr):
        N.lib().TSHip_InvalidateHostBuffer(C.c_void_p(ptr))

    @staticmethod
    def ClearHostBufferCache():
        N.lib().TSHip_ClearHostBufferCache()

    @staticmethod
    def SyncHostBuffer(array):
        """Copy the device copy kept for this host array (a KV cache the layer decode updates) back into it."""
        ok = N.lib().TSHip_SyncHostBuffer(C.c_void_p(array.ctypes.data), int(array.nbytes))
        N.check_result(ok, "sync_host_buffer")

    # -- MoE (GptOssModel.MoERoute / MoEForward twins, device tensors) --------------------------
    @staticmethod
    def MoERoute(logits, k):
        """logits [T x E] (CUDA fp32) -> (weights [T x k] fp32, ids [T x k] int32)."""
        torch = _torch()
        T = logits.shape[0]
        ids = torch.empty((T, k), dtype=torch.int32, device=logits.device)
        wts = torch.empty((T, k), dtype=torch.float32, device=logits.device)
        HipBasicOps.UseCurrentStream()
        ok = N.lib().TSHip_MoERouteF32Device(_device_view(logits), int(k), ids.data_ptr(), wts.data_ptr())
        N.check_result(ok, "moe_route")
        return wts, ids

    @staticmethod
    def MoEExpertsGptOssForward(hidden, ids, weights, gate_up_w, gate_up_b, down_w, down_b, ggml_type, n_experts, H, F,
                          alpha=1.702, limit=7.0):
        """Expert stage of GptOssModel.MoEForward for routed tokens; all tensors on the device."""
        torch = _torch()
        out = torch.empty((hidden.shape[0], H), dtype=torch.float32, device=hidden.device)
        HipBasicOps.UseCurrentStream()
        ok = N.lib().TSHip_MoEExpertsGptOssForwardF32Device(
            _device_view(out), _device_view(hidden), ids.data_ptr(), weights.data_ptr(), int(ids.shape[1]),
            gate_up_w.data_ptr(), None if gate_up_b is None else gate_up_b.data_ptr(), down_w.data_ptr(),
            None if down_b is None else down_b.data_ptr(), int(ggml_type), int(n_experts), int(H), int(F), float(alpha),
            float(limit))
        N.check_result(ok, "moe_experts_forward")
        return out

    # -- whole-layer decode (GgmlBasicOps.TransformerLayerDecode / TransformerModelDecode twins) ----
    @staticmethod
    def TransformerLayerDecode(hidden, attn_norm, qkv, q_norm, k_norm, o, ffn_norm, gate_up, down, k_cache, v_cache,
                               num_heads, num_kv_heads, head_dim, position, eps, rope_base, rope_freq_scale=1.0, rope_mode=2):
        """One token through one layer, in place on `hidden` [hidden_size] fp32.  Either everything is on the device (torch
        CUDA tensors, device QuantizedWeights; asynchronous on the current stream) or everything is in host memory (numpy
        arrays, host QuantizedWeights; weights, norms and KV caches are kept on the device under their host address, and
        SyncHostBuffer(k_cache) brings a cache back).  k_cache / v_cache fp32 [num_kv_heads, max_seq_len, head_dim];
        q_norm / k_norm may be None."""
        host = isinstance(hidden, np.ndarray)
        if host:
            fn = N.lib().TSHip_TransformerLayerDecode
        else:
            HipBasicOps.UseCurrentStream()
            fn = N.lib().TSHip_TransformerLayerDecodeDevice
        p = lambda t: None if t is None else HipBasicOps._addr(t)
        ok = fn(
            p(hidden), int(hidden.size if host else hidden.numel()), p(attn_norm),
            qkv.ptr, qkv.ggml_type, qkv.ne0, qkv.ne1, qkv.raw_bytes, p(q_norm), p(k_norm), int(head_dim),
            o.ptr, o.ggml_type, o.ne0, o.ne1, o.raw_bytes, p(ffn_norm),
            gate_up.ptr, gate_up.ggml_type, gate_up.ne0, gate_up.ne1, gate_up.raw_bytes,
            down.ptr, down.ggml_type, down.ne0, down.ne1, down.raw_bytes,
            p(k_cache), p(v_cache), int(num_heads), int(num_kv_heads), int(k_cache.shape[1]), int(position),
            float(eps), float(rope_base), float(rope_freq_scale), int(gate_up.ne1 // 2), int(rope_mode))
        N.check_result(ok, "transformer_layer_decode")

    @staticmethod
    def TransformerModelDecode(hidden, layers, num_heads, num_kv_heads, head_dim, position, eps, rope_base, rope_freq_scale=1.0,
                               rope_mode=2):
        """The same for a list of layers; each layer is a dict with the argument names of TransformerLayerDecode
        (attn_norm, qkv, q_norm, k_norm, o, ffn_norm, gate_up, down, k_cache, v_cache); shapes and types are shared.
        Host arrays or device tensors throughout, as for TransformerLayerDecode."""
        import ctypes as C
        host = isinstance(hidden, np.ndarray)
        if host:
            fn = N.lib().TSHip_TransformerModelDecode
        else:
            HipBasicOps.UseCurrentStream()
            fn = N.lib().TSHip_TransformerModelDecodeDevice
        n = len(layers)

        def arr(key, weight=False):
            vals = []
            for L in layers:
                t = L.get(key)
                vals.append(None if t is None else (t.ptr if weight else HipBasicOps._addr(t)))
            if all(v is None for v in vals):
                return None
            return (C.c_void_p * n)(*vals)
        l0 = layers[0]
        qkv, o, gu, dn = l0["qkv"], l0["o"], l0["gate_up"], l0["down"]
        ok = fn(
            HipBasicOps._addr(hidden), int(hidden.size if host else hidden.numel()), n, arr("attn_norm"), arr("qkv", True), arr("q_norm"), arr("k_norm"), arr("o", True),
            arr("ffn_norm"), arr("gate_up", True), arr("down", True), arr("k_cache"), arr("v_cache"),
            qkv.ggml_type, qkv.ne0, qkv.ne1, qkv.raw_bytes, o.ggml_type, o.ne0, o.ne1, o.raw_bytes,
            gu.ggml_type, gu.ne0, gu.ne1, gu.raw_bytes, dn.ggml_type, dn.ne0, dn.ne1, dn.raw_bytes,
            int(head_dim), int(num_heads), int(num_kv_heads), int(l0["k_cache"].shape[1]), int(position), float(eps),
            float(rope_base), float(rope_freq_scale), int(gu.ne1 // 2), int(rope_mode))
        N.check_result(ok, "transformer_model_decode")

    # -- many sequences: rotary positions, a paged cache, attention over its pages, sampling (device tensors) ------------
    @staticmethod
    def RoPE(result, input, positions, rope):
        """result[t, h] = input[t, h] turned by positions[t]: [tokens, heads, head_dim] float32 device tensors (result may be input), positions
        int32 [tokens], rope a RotaryPositions."""
        rv, iv = _device_view3(result, "RoPE"), _device_view3(input, "RoPE")
        device = input.get_device()
        if result.get_device() != device:
            raise ValueError("RoPE requires tensors in GPU memory of one device.")
        if rope.device is not None and rope.device != device:
            rope._elsewhere()
        pos = _vector(positions, _torch().int32, iv.dim0, "positions", device)
        _use_stream_of(device)
        ok = N.lib().TSHip_RoPEF32Device(rv, iv, pos, rope.ref)
        N.check_result(ok, "rope")

    @staticmethod
    def RoPEStorePaged(query, qkv, cache, row_starts, context_lens, rope, q_norm=None, k_norm=None, eps=1e-6, positions=None):
        """From a fused QKV projection to the attention over a PagedKVCache: rows row_starts[s] .. row_starts[s + 1] - 1 of qkv [rows, (heads +
        2 kv heads) head_dim] are the last tokens of the context_lens[s] of sequence s.  q and k heads are normed (q_norm / k_norm
        [head_dim], None: not) and turned by their position in the sequence (or positions[row]); q goes to query [rows, heads
        head_dim], k and v into the cache."""
        torch = _torch()
        f32, i32 = torch.float32, torch.int32
        qv, xv = _device_view(query), _device_view(qkv)
        dim, device = cache.head_dim, cache.device
        starts, lens = cache._sequences(row_starts, context_lens, i32)
        if rope.device is not None and rope.device != device:
            rope._elsewhere()
        pos = _vector(positions, i32, xv.dim0, "positions", device)
        qn, kn = _vector(q_norm, f32, dim, "q_norm", device), _vector(k_norm, f32, dim, "k_norm", device)
        if query.get_device() != device or qkv.get_device() != device:
            raise ValueError("query and qkv must be on the device of the cache.")
        _use_stream_of(device)
        ok = N.lib().TSHip_RoPEStorePagedF32Device(qv, xv, qv.dim1 // dim, cache.ref, starts, lens, pos, qn, kn, eps, rope.ref)
        N.check_result(ok, "rope_store_paged")

    @staticmethod
    def ResizeSequences(pool, lengths, moves, missing):
        """Sequences of a PagePool become lengths[s] tokens long (int32; negative: stay as they are; 0: have no pages).  Shorter ones give back the pages behind their
        ends first, longer ones get the lowest free pages; one that goes on in a begun page which others have too gets a page in its place, and moves
        [sequences, 2] int32 lists the copies (from, to) for CopyPages, -1 behind the last.  Where the free pages do not suffice none grows, and missing [1] int32 says
        how many more it takes (else 0)."""
        i32 = _torch().int32
        to = _vector(lengths, i32, pool.num_seqs, "lengths", pool.device)
        if to is None or missing is None:
            raise ValueError("ResizeSequences requires lengths and missing.")
        m, short = pool._moves(moves, pool.num_seqs), _vector(missing, i32, 1, "missing", pool.device)
        _use_stream_of(pool.device)
        N.check_result(N.lib().TSHip_ResizeSequencesDevice(pool.ref, to, m, short), "resize_sequences")

    @staticmethod
    def ForkSequences(pool, children, parents, moves, missing):
        """Sequences children[i] of a PagePool become what parents[i] were before the call (int32; of pairs with one child the last counts): they give back their
        pages and share the whole ones of their parents.  One of those that have a begun page keeps it (the parent, else the lowest child), the others get copies in
        free pages, listed in moves [pairs, 2] as in ResizeSequences.  Where the free pages do not suffice nothing changes, and missing [1] says how many more it takes."""
        i32 = _torch().int32
        if children is None or parents is None or missing is None:
            raise ValueError("ForkSequences requires children, parents and missing.")
        count = children.numel()
        c, p = _vector(children, i32, count, "children", pool.device), _vector(parents, i32, count, "parents", pool.device)
        m, short = pool._moves(moves, count), _vector(missing, i32, 1, "missing", pool.device)
        _use_stream_of(pool.device)
        N.check_result(N.lib().TSHip_ForkSequencesDevice(pool.ref, c, p, count, m, short), "fork_sequences")

    @staticmethod
    def CompactPages(pool, moves):
        """Used pages of a PagePool move to the front: the last ones into the lowest free ones, as many as moves [room, 2] int32 has room for; it lists the
        copies (from, to) for CopyPages, -1 behind the last."""
        m = pool._moves(moves, None)
        _use_stream_of(pool.device)
        N.check_result(N.lib().TSHip_CompactPagesDevice(pool.ref, m, moves.shape[0]), "compact_pages")

    @staticmethod
    def CopyPages(dst, src, moves):
        """Pages moves[i, 0] of the PagedKVCache src go into pages moves[i, 1] of dst (int32 [moves, 2]; a pair outside the pages, as -1 is, is left out): one cache
        or two of one page size, number of heads and head_dim, of one type or two (rounded as RoPEStorePaged does).  No page that is written may be in another pair."""
        if src.device != dst.device:
            raise ValueError("CopyPages requires caches on one device.")
        m = _pairs(moves, None, dst.device)
        _use_stream_of(dst.device)
        N.check_result(N.lib().TSHip_CopyPagesDevice(dst.ref, src.ref, m, moves.shape[0]), "copy_pages")

    @staticmethod
    def PagedAttention(result, query, cache, row_starts, context_lens, scale, window=0, sinks=None, first=0):
        """Attention of the sequences' new tokens (rows as in RoPEStorePaged) over a PagedKVCache that holds their keys and values already:
        each sees the positions up to its own, the last `window` of them (0: all) and, of those before, the first `first` of the sequence.  query and result [rows, heads head_dim]
        float32 (may be one tensor); sinks [heads] float32: logits that take part in the softmax and carry no value."""
        if not -2 ** 31 <= window < 2 ** 31:         # (the call takes 32 bits of it)
            raise ValueError("PagedAttention requires a window below 2^31.")
        if not 0 <= first < 2 ** 31:
            raise ValueError("PagedAttention requires a number of first positions from 0 to below 2^31.")
        torch = _torch()
        rv, qv = _device_view(result), _device_view(query)
        heads, device = qv.dim1 // cache.head_dim, cache.device
        starts, lens = cache._sequences(row_starts, context_lens, torch.int32)
        extra = _vector(sinks, torch.float32, heads, "sinks", device)
        if query.get_device() != device or result.get_device() != device:
            raise ValueError("query and result must be on the device of the cache.")
        _use_stream_of(device)
        if first:
            ok = N.lib().TSHip_PagedAttentionFirstF32Device(rv, qv, heads, cache.ref, starts, lens, scale, window, first, extra)
        else:
            ok = N.lib().TSHip_PagedAttentionF32Device(rv, qv, heads, cache.ref, starts, lens, scale, window, extra)
        N.check_result(ok, "paged_attention")

    @staticmethod
    def SampleTokens(tokens, logits, uniforms, temperature, top_k=None, top_p=None, min_p=None, probabilities=None):
        """tokens[r] (int32) drawn from logits [rows, vocab] (float32): e^(l / temperature[r]) of the top_k[r] (int32) likeliest, of these the
        fewest that reach top_p[r], of these those with min_p[r] of the likeliest's weight; the first in index order whose
        cumulated weight exceeds uniforms[r] of the total.  temperature 0: the likeliest.  None: no such limit.  probabilities
        [rows] float32: of the tokens drawn."""
        torch = _torch()
        lv = _device_view(logits)
        rows, device = lv.dim0, logits.get_device()
        f32, i32 = torch.float32, torch.int32
        if tokens is None or uniforms is None or temperature is None:
            raise ValueError("SampleTokens requires tokens, uniforms and temperature.")
        u, t = _vector(uniforms, f32, rows, "uniforms", device), _vector(temperature, f32, rows, "temperature", device)
        k, p, m = _vector(top_k, i32, rows, "top_k", device), _vector(top_p, f32, rows, "top_p", device), _vector(min_p, f32, rows, "min_p", device)
        out, probs = _vector(tokens, i32, rows, "tokens", device), _vector(probabilities, f32, rows, "probabilities", device)
        _use_stream_of(device)
        N.check_result(N.lib().TSHip_SampleTokensF32Device(lv, u, t, k, p, m, out, probs), "sample_tokens")

    # -- LinearForward twin (ModelBase.cs:875-905): allocate result, route by residency -----
    @staticmethod
    def LinearForward(m1, qw: QuantizedWeight):
        if qw.is_device:
            torch = _torch()
            result = torch.empty((m1.shape[0], qw.ne1), dtype=torch.float32, device=m1.device)
            HipBasicOps.UseCurrentStream()
            HipBasicOps.AddmmQuantDevice(result, m1, qw.ptr, qw.ggml_type, qw.ne0, qw.ne1, qw.raw_bytes)
            return result
        result = np.empty((m1.shape[0], qw.ne1), dtype=np.float32)
        HipBasicOps.AddmmQuant(result, m1, qw.ptr, qw.ggml_type, qw.ne0, qw.ne1, qw.raw_bytes)
        return result

    @staticmethod
    def UseCurrentStream():
        """Launch the *Device entry points on torch's current stream."""
        torch = _torch()
        try:                                    # current_stream().cuda_stream without the stream object
            handle = torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice()) if torch.cuda.is_initialized() else None
        except AttributeError:                  # (private names, which a torch build may lack)
            handle = None
        if handle is None:
            handle = torch.cuda.current_stream().cuda_stream
        N.lib().TSHip_SetStream(handle)
