"""Torch-facing wrappers over the C ABI: allocate outputs/scratch with torch, pass raw pointers.

These functions are what the drop-in modules and the `quant_linear_cuda` / `quant_embedding_cuda` /
`fast_hadamard_transform_cuda` stand-ins call.  All of them require CUDA tensors; there is no fallback.
"""
from __future__ import annotations

import ctypes
import math

import torch

from ._lib import Prefetch, Proj, check, lib, torch_ext

_DTYPE_CODE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}

_scratch: dict = {}      # (device index, stream handle) -> uint8 tensor whose counter region is zero
_status: dict = {}       # device index -> int32[1] status word


def _stream_handle(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def status_word(device: torch.device) -> torch.Tensor:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    t = _status.get(idx)
    if t is None:
        ext = torch_ext()
        # one word per device, shared with the torch binding when that is loaded
        t = ext.status_tensor(idx) if ext is not None else torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", idx))
        _status[idx] = t
    return t


def read_and_clear_status(device) -> int:
    """Synchronising read of the kernel diagnostics word (bit 0: an embedding id was out of range; bit 1: a bounded
    wait gave up; bit 2: a slicing index was outside the source layer, or a slot or page outside the KV cache, or bounds of
    packed rows named rows that do not exist; bit 3: a page plan ran out of free pages or of columns of the block table)."""
    t = status_word(torch.device(device))
    v = int(t.item())
    t.zero_()
    return v


def _scratch_for(device: torch.device, nbytes: int) -> torch.Tensor:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    key = (idx, _stream_handle(device))
    buf = _scratch.get(key)
    if buf is None or buf.numel() < nbytes:
        size = max(nbytes, 1 << 20)
        size = (size + (1 << 20) - 1) >> 20 << 20
        buf = torch.zeros(size, dtype=torch.uint8, device=torch.device("cuda", idx))
        _scratch[key] = buf
    return buf


def _require_cuda(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (uniql_b200 has no CPU path)")


_need_cache: dict = {}   # (m, n, k, hadamard_dim) -> scratch bytes


def w4a16_linear(x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None,
                 n_out: int, hadamard_dim: int = 0, out: torch.Tensor | None = None, comm=None) -> torch.Tensor:
    """y[m, n_out] = x[m, k] @ dequant(weight, scale)[:, :n_out] (+ bias); x fp16 2-D, row-major.
    With `comm` (a communicator handle from uniql_comm_create) the result is summed over the ranks inside the
    kernel (row-parallel linear, m <= 16)."""
    if not (x.is_cuda and weight.is_cuda and scale.is_cuda):
        raise RuntimeError("x, weight and scale must be CUDA tensors (uniql_b200 has no CPU path)")
    if x.dtype != torch.float16 or x.dim() != 2:
        raise RuntimeError("x must be a 2-D float16 tensor")
    if weight.dtype != torch.int32 or scale.dtype != torch.float16:
        raise RuntimeError("weight must be int32 and scale float16")
    if x.stride(1) != 1:
        x = x.contiguous()
    m, k = x.shape
    kt, n2 = weight.shape
    if kt * 16 != k:
        raise RuntimeError(f"size_k mismatch: x has {k} columns, packed weight covers {kt * 16}")
    n = n2 // 2
    groups = scale.shape[0]
    if groups == 1 and k != 128:
        groupsize = -1
    else:
        if k % groups != 0:
            raise RuntimeError("scale rows do not divide k")
        groupsize = k // groups
    if scale.shape[1] != n:
        raise RuntimeError("scale width does not match the packed weight")
    if not weight.is_contiguous() or not scale.is_contiguous():
        raise RuntimeError("weight and scale must be contiguous")
    bias_ptr = None
    if bias is not None:
        if bias.dtype != torch.float16 or bias.numel() < n_out or not bias.is_contiguous():
            raise RuntimeError("bias must be a contiguous float16 tensor with at least n_out elements")
        bias_ptr = bias.data_ptr()
    if (m > 1 and x.stride(0) % 8 != 0) or x.data_ptr() % 16 != 0:
        x = x.clone(memory_format=torch.contiguous_format)
    lda = x.stride(0) if m > 1 else k
    dev = x.device
    idx = dev.index
    switch = torch.cuda.current_device() != idx
    if switch:
        prev = torch.cuda.current_device()
        torch.cuda.set_device(idx)
    try:
        if out is None:
            out = torch.empty((m, n_out), dtype=torch.float16, device=dev)
        L = lib()
        key = (m, n, k, hadamard_dim)
        nbytes = _need_cache.get(key)
        if nbytes is None:
            nbytes = _need_cache[key] = L.uniql_w4a16_scratch_bytes(m, n, k, hadamard_dim)
        stream = torch._C._cuda_getCurrentRawStream(idx)
        skey = (idx, stream)
        scratch = _scratch.get(skey)
        if scratch is None or scratch.numel() < nbytes:
            scratch = _scratch_for(dev, nbytes)
        st = _status.get(idx)
        if st is None:
            st = status_word(dev)
        if comm is not None:
            code = L.uniql_w4a16_linear_allreduce(
                comm, x.data_ptr(), lda, weight.data_ptr(), scale.data_ptr(), bias_ptr,
                out.data_ptr(), out.stride(0), m, n, n_out, k, groupsize,
                scratch.data_ptr(), scratch.numel(), st.data_ptr(), stream)
        else:
            code = L.uniql_w4a16_linear(
                x.data_ptr(), lda, weight.data_ptr(), scale.data_ptr(), bias_ptr,
                out.data_ptr(), out.stride(0), m, n, n_out, k, groupsize, hadamard_dim,
                scratch.data_ptr(), scratch.numel(), st.data_ptr(), stream)
    finally:
        if switch:
            torch.cuda.set_device(prev)
    if code != 0:
        check(code, "uniql_w4a16_linear")
    return out


_EPILOGUES = {"none": 0, "swiglu": 1}
TP_REDUCE, TP_GATHER_OUT, TP_GATHER_IN = 1, 2, 4
_group_need_cache: dict = {}


def w4a16_linear_group(x: torch.Tensor | None, layers, epilogue: str = "none", residual: torch.Tensor | None = None,
                       hadamard_dim: int = 0, outs=None, comm=None, tp_flags: int = 0, col_offset: int = 0,
                       k_offset: int = 0, m: int | None = None, prefetch=None):
    """One launch for up to four projections that read the same activations: all options below for m <= 16 (on the
    decode kernel or the operand-swapped tensor-core kernel, whichever is faster), plain outputs for 17 <= m <= 128.

    layers: sequence of (weight int32 [k/16, 2n], scale fp16 [k/128, n], bias fp16 or None, n_out).
    epilogue "swiglu": two layers (gate, up) -> one output silu(gate) * up.  residual: fp16 [m, n_out] added to the
    result (single layer or swiglu).  hadamard_dim: size of the Hadamard transform applied to the rows of x first.
    With `comm` (communicator handle) and tp_flags (TP_REDUCE / TP_GATHER_OUT / TP_GATHER_IN) the launch is a step of a
    tensor-parallel layer; with TP_GATHER_IN x may be None and m must be given.
    prefetch: up to four tensors (or (tensor, bytes) pairs) -- the packed weights the following launches will stream --
    that the kernel asks L2 for when its own stream ends.
    Returns the list of outputs (one tensor for swiglu)."""
    if epilogue not in _EPILOGUES:
        raise RuntimeError(f"unknown epilogue {epilogue!r}")
    layers = list(layers)
    w0 = layers[0][0]
    if not w0.is_cuda:
        raise RuntimeError("weights must be CUDA tensors (uniql_b200 has no CPU path)")
    dev = w0.device
    k = w0.shape[0] * 16
    if x is not None:
        if not x.is_cuda or x.dtype != torch.float16 or x.dim() != 2:
            raise RuntimeError("x must be a 2-D float16 CUDA tensor")
        if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) % 8 != 0) or x.data_ptr() % 16 != 0:
            x = x.contiguous() if x.stride(1) != 1 else x.clone(memory_format=torch.contiguous_format)
        m = x.shape[0]
        if x.shape[1] != k:
            raise RuntimeError(f"size_k mismatch: x has {x.shape[1]} columns, packed weight covers {k}")
        lda = x.stride(0) if m > 1 else k
        x_ptr = x.data_ptr()
    else:
        if not (tp_flags & TP_GATHER_IN) or m is None:
            raise RuntimeError("x may only be omitted for a TP_GATHER_IN launch with m given")
        lda, x_ptr = k, None
    n_outputs = 1 if epilogue == "swiglu" else len(layers)
    if outs is None:
        outs = [torch.empty((m, layers[i][3]), dtype=torch.float16, device=dev) for i in range(n_outputs)]
    arr = (Proj * len(layers))()
    ns = (ctypes.c_int64 * len(layers))()
    for i, (w, s, b, n_out) in enumerate(layers):
        if w.dtype != torch.int32 or s.dtype != torch.float16 or not w.is_contiguous() or not s.is_contiguous():
            raise RuntimeError("weight must be contiguous int32 and scale contiguous float16")
        if w.shape[0] * 16 != k or s.shape[0] * 128 != k or s.shape[1] * 2 != w.shape[1]:
            raise RuntimeError("projections of one launch must share k, with group-128 scales")
        if b is not None and (b.dtype != torch.float16 or b.numel() < n_out or not b.is_contiguous()):
            raise RuntimeError("bias must be a contiguous float16 tensor with at least n_out elements")
        d = outs[min(i, n_outputs - 1)]
        arr[i].B, arr[i].s = w.data_ptr(), s.data_ptr()
        arr[i].bias = b.data_ptr() if b is not None else None
        arr[i].D, arr[i].ldd = d.data_ptr(), d.stride(0)
        arr[i].n, arr[i].n_out = s.shape[1], n_out
        ns[i] = s.shape[1]
    res_ptr, ldr = None, 0
    if residual is not None:
        if residual.dtype != torch.float16 or residual.dim() != 2 or residual.stride(1) != 1:
            raise RuntimeError("residual must be a 2-D float16 tensor with unit column stride")
        res_ptr, ldr = residual.data_ptr(), residual.stride(0)
    pf_arr, npf = None, 0
    if prefetch:
        pf_arr = (Prefetch * 4)()
        for item in prefetch:
            t, nb = item if isinstance(item, tuple) else (item, item.numel() * item.element_size())
            if npf < 4 and nb >= 128:
                pf_arr[npf].ptr, pf_arr[npf].bytes = t.data_ptr(), min(nb, t.numel() * t.element_size())
                npf += 1
    idx = dev.index
    L = lib()
    with torch.cuda.device(dev):
        key = (m, k, tuple(ns), _EPILOGUES[epilogue], hadamard_dim)
        nbytes = _group_need_cache.get(key)
        if nbytes is None:
            nbytes = _group_need_cache[key] = L.uniql_w4a16_group_scratch_bytes(m, k, ns, len(layers), _EPILOGUES[epilogue],
                                                                                 hadamard_dim)
        scratch = _scratch_for(dev, nbytes)
        st = status_word(dev)
        stream = torch._C._cuda_getCurrentRawStream(idx)
        if comm is not None:
            code = L.uniql_w4a16_linear_group_tp(comm, tp_flags, col_offset, k_offset, x_ptr, lda, m, k, arr, len(layers),
                                                 _EPILOGUES[epilogue], res_ptr, ldr, hadamard_dim, pf_arr, npf,
                                                 scratch.data_ptr(), scratch.numel(), st.data_ptr(), stream)
        else:
            code = L.uniql_w4a16_linear_group(x_ptr, lda, m, k, arr, len(layers), _EPILOGUES[epilogue], res_ptr, ldr,
                                              hadamard_dim, pf_arr, npf, scratch.data_ptr(), scratch.numel(),
                                              st.data_ptr(), stream)
    if code != 0:
        check(code, "uniql_w4a16_linear_group")
    return outs


def w4_embedding(ids: torch.Tensor, weight: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """out[..., :] = dequantised rows of the 4-bit table for int64 ids of shape [T] or [B, T]."""
    _require_cuda(ids, "input"); _require_cuda(weight, "weight"); _require_cuda(scales, "scale")
    if weight.dim() != 2 or weight.dtype != torch.int32:
        raise RuntimeError("weight must be a 2-D int32 tensor")
    if scales.dim() != 1 or scales.dtype != torch.float16 or scales.numel() != weight.shape[0]:
        raise RuntimeError("scale must be a 1-D float16 tensor with one entry per table row")
    if ids.dim() not in (1, 2) or ids.dtype != torch.int64:
        raise RuntimeError("input must be a 1-D or 2-D int64 tensor")
    ids_c = ids.contiguous()
    weight = weight.contiguous()
    vocab, words = weight.shape
    dim = words * 8
    out = torch.empty((*ids.shape, dim), dtype=torch.float16, device=ids.device)
    with torch.cuda.device(ids.device):
        code = lib().uniql_w4_embedding(
            ids_c.data_ptr(), ids_c.numel(), weight.data_ptr(), scales.contiguous().data_ptr(), out.data_ptr(),
            vocab, dim, status_word(ids.device).data_ptr(), _stream_handle(ids.device))
    check(code, "uniql_w4_embedding")
    return out


def hadamard(x: torch.Tensor, scale: float) -> torch.Tensor:
    """New tensor y = H x * scale along the last axis (x is made contiguous first)."""
    _require_cuda(x, "x")
    if x.dtype not in _DTYPE_CODE:
        raise RuntimeError(f"unsupported dtype {x.dtype}")
    xc = x.contiguous()
    dim = xc.shape[-1]
    rows = xc.numel() // dim if dim else 0
    y = torch.empty_like(xc)
    with torch.cuda.device(x.device):
        code = lib().uniql_hadamard(xc.data_ptr(), y.data_ptr(), rows, dim, float(scale), _DTYPE_CODE[x.dtype],
                                    _stream_handle(x.device))
    check(code, "uniql_hadamard")
    return y


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up for fp16 CUDA tensors of the same shape, one pass (fp16 SiLU, fp16 product, as the two PyTorch
    ops would round)."""
    _require_cuda(gate, "gate"); _require_cuda(up, "up")
    if gate.dtype != torch.float16 or up.dtype != torch.float16 or gate.shape != up.shape:
        raise RuntimeError("gate and up must be float16 tensors of the same shape")
    cols = gate.shape[-1]
    g2, u2 = gate.reshape(-1, cols), up.reshape(-1, cols)
    if g2.stride(1) != 1 or g2.stride(0) % 8 or g2.data_ptr() % 16:
        g2 = g2.contiguous()
    if u2.stride(1) != 1 or u2.stride(0) % 8 or u2.data_ptr() % 16:
        u2 = u2.contiguous()
    out = torch.empty(g2.shape, dtype=torch.float16, device=gate.device)
    with torch.cuda.device(gate.device):
        code = lib().uniql_silu_mul(g2.data_ptr(), g2.stride(0), u2.data_ptr(), u2.stride(0), out.data_ptr(), cols,
                                    g2.shape[0], cols, _stream_handle(gate.device))
    check(code, "uniql_silu_mul")
    return out.view(gate.shape)


def hadamard_base_matrix(base: int) -> torch.Tensor:
    """The int8 [base, base] matrix of +1 / -1 the library applies for orders 12, 20, 28 and 40 right now."""
    import ctypes
    buf = (ctypes.c_int8 * (base * base))()
    check(lib().uniql_hadamard_base_matrix(int(base), buf), "uniql_hadamard_base_matrix")
    return torch.tensor(list(buf), dtype=torch.int8).reshape(base, base)


def hadamard_set_base_matrix(base: int, matrix=None) -> None:
    """Replace the order-`base` Hadamard matrix (12, 20, 28, 40) for every transform launched afterwards in this
    process; `matrix` is a [base, base] array of +1 / -1 with orthogonal rows, None restores the built-in one.  The
    reference's transforms come from the third-party fast_hadamard_transform package (quantize/hadamard_helpers.py:18-36):
    passing that package's tables here makes this library reproduce them."""
    import ctypes
    if matrix is None:
        check(lib().uniql_hadamard_set_base_matrix(int(base), None), "uniql_hadamard_set_base_matrix")
        return
    m = torch.as_tensor(matrix).to(torch.int8).contiguous().cpu()
    if tuple(m.shape) != (base, base):
        raise RuntimeError(f"matrix must be [{base}, {base}]")
    buf = (ctypes.c_int8 * (base * base))(*m.reshape(-1).tolist())
    check(lib().uniql_hadamard_set_base_matrix(int(base), buf), "uniql_hadamard_set_base_matrix")


def w4a16_quantize(weight: torch.Tensor, group_scale: torch.Tensor | None = None, n_pad: int | None = None,
                   want_ref: bool = True):
    """Quantise and pack an nn.Linear weight [out, in] (fp16, CUDA) on the GPU.

    Returns (w_ref fp16 [Kp, n_pad] or None, packed int32 [Kp/16, 2*n_pad], scales fp16 [Kp/128, n_pad]) with the
    values of the reference's w4a16_quantize(weight.T, 4, 128, group_scale, pad_out) (quantize_helpers.py:184-241);
    n_pad defaults to `out` rounded up to 256 as in W4A16B16O16Linear.from_fp16 (quant_linear_layers.py:65-66)."""
    _require_cuda(weight, "weight")
    if weight.dim() != 2:
        raise RuntimeError("weight must be [out_features, in_features]")
    w = weight.detach()
    if w.dtype != torch.float16:
        w = w.to(torch.float16)
    if w.stride(1) != 1:
        w = w.contiguous()
    n_out, k_in = w.shape
    if n_pad is None:
        n_pad = (n_out + 255) // 256 * 256
    kp = (k_in + 127) // 128 * 128
    gs = None
    if group_scale is not None:
        _require_cuda(group_scale, "group_scale")
        gs = group_scale.detach().to(torch.float16).contiguous()
        if tuple(gs.shape) != (kp // 128, n_out):
            raise RuntimeError(f"group_scale must be [{kp // 128}, {n_out}], got {tuple(gs.shape)}")
    dev = w.device
    packed = torch.empty((kp // 16, 2 * n_pad), dtype=torch.int32, device=dev)
    scales = torch.empty((kp // 128, n_pad), dtype=torch.float16, device=dev)
    w_ref = torch.empty((kp, n_pad), dtype=torch.float16, device=dev) if want_ref else None
    with torch.cuda.device(dev):
        code = lib().uniql_w4a16_quantize(w.data_ptr(), w.stride(0), n_out, k_in,
                                          gs.data_ptr() if gs is not None else None,
                                          packed.data_ptr(), scales.data_ptr(),
                                          w_ref.data_ptr() if w_ref is not None else None, n_pad,
                                          _stream_handle(dev))
    check(code, "uniql_w4a16_quantize")
    return w_ref, packed, scales


def w4a16_gather_columns(weight: torch.Tensor, scale: torch.Tensor, col_index: torch.Tensor, n_out_pad: int,
                         zero_rows_from: int | None = None):
    """New packed layer with output column c = source column col_index[c], zero-padded to n_out_pad columns; rows from
    `zero_rows_from` on get code 0.  Returns (packed int32 [K/16, 2*n_out_pad], scales fp16 [K/128, n_out_pad])."""
    _require_cuda(weight, "weight")
    _require_cuda(scale, "scale")
    dev = weight.device
    size_k, n_src_pad = weight.shape[0] * 16, weight.shape[1] // 2
    # the CPU path would raise IndexError here too (negative entries are allowed: they produce zero columns); an index that
    # is still on the host is checked there, one on the GPU costs a synchronisation
    idx = col_index.to(dtype=torch.int32)
    if idx.numel() and int(idx.max()) >= n_src_pad:
        raise RuntimeError("col_index out of range")
    idx = idx.to(device=dev).contiguous()
    weight, scale = weight.contiguous(), scale.contiguous()
    packed = torch.empty((size_k // 16, 2 * n_out_pad), dtype=torch.int32, device=dev)
    scales = torch.empty((size_k // 128, n_out_pad), dtype=torch.float16, device=dev)
    with torch.cuda.device(dev):
        code = lib().uniql_w4a16_gather_columns(weight.data_ptr(), scale.data_ptr(), size_k, n_src_pad, idx.data_ptr(),
                                                idx.numel(), size_k if zero_rows_from is None else zero_rows_from,
                                                packed.data_ptr(), scales.data_ptr(), n_out_pad,
                                                status_word(dev).data_ptr(), _stream_handle(dev))
    check(code, "uniql_w4a16_gather_columns")
    return packed, scales


def w4a16_dequantize_rows(weight: torch.Tensor, scale: torch.Tensor, row_index: torch.Tensor, n_real: int) -> torch.Tensor:
    """fp16 [n_real, len(row_index)]: dequantised weights of the chosen input rows in nn.Linear layout."""
    _require_cuda(weight, "weight")
    _require_cuda(scale, "scale")
    dev = weight.device
    size_k, n_src_pad = weight.shape[0] * 16, weight.shape[1] // 2
    idx = row_index.to(dtype=torch.int32)
    if idx.numel() and (int(idx.min()) < 0 or int(idx.max()) >= size_k):
        raise RuntimeError("row_index out of range")
    idx = idx.to(device=dev).contiguous()
    weight, scale = weight.contiguous(), scale.contiguous()
    out = torch.empty((n_real, idx.numel()), dtype=torch.float16, device=dev)
    with torch.cuda.device(dev):
        code = lib().uniql_w4a16_dequantize_rows(weight.data_ptr(), scale.data_ptr(), size_k, n_src_pad, idx.data_ptr(),
                                                 idx.numel(), n_real, out.data_ptr(), idx.numel(),
                                                 status_word(dev).data_ptr(), _stream_handle(dev))
    check(code, "uniql_w4a16_dequantize_rows")
    return out


# ---- attention around a paged KV cache held in 4 bits (layout and rules: include/uniql_b200.h) ---------------------------
# They go through the torch binding like the modules' forward; with UNIQL_B200_TORCH_EXT=0 the same C calls are made over ctypes.

def _ints(t: torch.Tensor, like: torch.Tensor, dim: int, name: str) -> torch.Tensor:
    if not t.is_cuda or t.dtype != torch.int32 or t.dim() != dim:
        raise RuntimeError(f"{name} must be a {dim}-D int32 CUDA tensor")
    if t.device != like.device:
        raise RuntimeError(f"{name} is on another device")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise RuntimeError(f"{name} must have unit stride in its last dimension")
    return t


def _ld(table: torch.Tensor) -> int:
    if table.shape[0] > 1 and table.stride(0) < table.shape[1]:
        raise RuntimeError("rows of block_table must not overlap")
    return table.stride(0) if table.shape[0] > 1 else table.shape[1]


def _cache_shape(codes: torch.Tensor, scales: torch.Tensor):
    if not codes.is_cuda or not scales.is_cuda:
        raise RuntimeError("codes and scales must be CUDA tensors (uniql_b200 has no CPU path)")
    if codes.dtype != torch.int32 or scales.dtype != torch.float16:
        raise RuntimeError("codes must be int32 and scales float16")
    if codes.dim() != 5 or codes.shape[1] != 2 or not codes.is_contiguous():
        raise RuntimeError("codes must be a contiguous [pages, 2, kv_heads, page_size, words] tensor")
    if scales.shape != (*codes.shape[:4], 2) or not scales.is_contiguous() or scales.device != codes.device:
        raise RuntimeError("scales must be a contiguous [pages, 2, kv_heads, page_size, 2] tensor of the same cache")
    pages, _, heads, page, words = codes.shape
    return pages, heads, page, words * 8


def _kv_dtype(t: torch.Tensor, name: str) -> int:
    if t.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"{name} must be float16 or bfloat16")
    return _DTYPE_CODE[t.dtype]


def _head_rows(x: torch.Tensor) -> torch.Tensor:
    ok = x.stride(2) == 1 and x.data_ptr() % 16 == 0 and all(x.shape[i] <= 1 or (x.stride(i) > 0 and x.stride(i) % 8 == 0) for i in (0, 1))
    return x if ok else x.clone(memory_format=torch.contiguous_format)


def _row_strides(x: torch.Tensor):
    return (x.stride(0) if x.shape[0] > 1 else x.shape[1] * x.shape[2]), (x.stride(1) if x.shape[1] > 1 else x.shape[2])


def kv4_cache(num_pages: int, kv_heads: int, page_size: int, head_dim: int, device="cuda"):
    """(codes, scales) of an empty cache of one layer; head_dim: the larger of K's and V's head size."""
    if page_size not in (16, 32, 64, 128, 256) or not 0 < head_dim <= 128 or head_dim % 8:
        raise RuntimeError("page_size must be 16, 32, 64, 128 or 256 and head_dim a multiple of 8 up to 128")
    words = (64 if head_dim <= 64 else 128) // 8
    return (torch.zeros(num_pages, 2, kv_heads, page_size, words, dtype=torch.int32, device=device),
            torch.zeros(num_pages, 2, kv_heads, page_size, 2, dtype=torch.float16, device=device))


def kv_page_plan(lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                 free_count: torch.Tensor, page_size: int, total_new: int, in_place: bool = False, whole: bool = False):
    """What a step's new tokens need, worked out on the GPU from the requests' lengths: pages from the top of the stack
    `free_pages` (free_count[0] of them are left) go into `block_table` in place.  Returns (slots int64 [total_new], positions
    int64 [total_new], cu_new int32 [batch + 1], lens after the step, free_count after the step); with in_place the last two are
    `lens` and `free_count` themselves.  total_new: places to fill (the rows of the step's tensors; those behind the last
    token get slot -1).  A shortage of pages or of table columns gives slots of -1 and status bit 3.  With `whole` a request that
    cannot have all its pages, columns and places is left out of the step (its length and table row stay, its slots are -1), and two
    more results say what the step attends to: its requests' keys (int32 [batch], 0 for one left out) and their exclusive sums
    (int32 [batch + 1]).  The results may share one storage."""
    ext = torch_ext()
    if ext is not None:
        return tuple(ext.kv_page_plan(lens, new_lens, block_table, free_pages, free_count, page_size, total_new, in_place, whole))
    for t, dim, name in ((lens, 1, "lens"), (new_lens, 1, "new_lens"), (block_table, 2, "block_table"), (free_pages, 1, "free_pages"),
                         (free_count, 1, "free_count")):
        _ints(t, lens, dim, name)
    batch = lens.shape[0]
    if new_lens.shape[0] != batch or block_table.shape[0] != batch:
        raise RuntimeError("lens, new_lens and block_table must have one row per request")
    if free_count.shape[0] != 1 or total_new < 0:
        raise RuntimeError("free_count must have one entry and total_new must not be negative")
    ld, dev = _ld(block_table), lens.device
    slots = torch.empty(total_new, dtype=torch.int64, device=dev)
    positions = torch.empty(total_new, dtype=torch.int64, device=dev)
    cu = torch.empty(batch + 1, dtype=torch.int32, device=dev)
    lens_out = lens if in_place else torch.empty_like(lens)
    count_out = free_count if in_place else torch.empty_like(free_count)
    keys = (torch.empty(batch, dtype=torch.int32, device=dev), torch.empty_like(cu)) if whole else ()
    name = "uniql_kv_step_plan" if whole else "uniql_kv_page_plan"
    with torch.cuda.device(dev):
        code = getattr(lib(), name)(lens.data_ptr(), new_lens.data_ptr(), batch, block_table.data_ptr(), ld, block_table.shape[1],
                                    free_pages.data_ptr(), free_pages.shape[0], free_count.data_ptr(), page_size, total_new,
                                    slots.data_ptr(), positions.data_ptr(), cu.data_ptr(), lens_out.data_ptr(), count_out.data_ptr(),
                                    *(t.data_ptr() for t in keys), status_word(dev).data_ptr(), _stream_handle(dev))
    check(code, name)
    return slots, positions, cu, lens_out, count_out, *keys


def kv4_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor) -> None:
    """Quantise the rows k, v [tokens, kv_heads, channels] (fp16 or bf16) to 4 bits with one scale and zero per token and head and
    store them in the cache at `slots` (int64; -1 skips the token; the others must differ)."""
    ext = torch_ext()
    if ext is not None:
        ext.kv4_append(k, v, slots, codes, scales)
        return
    pages, heads, page, dp = _cache_shape(codes, scales)
    if not k.is_cuda or not v.is_cuda or k.dim() != 3 or v.dim() != 3:
        raise RuntimeError("k and v must be [tokens, kv_heads, channels] CUDA tensors")
    dtype = _kv_dtype(k, "k")
    if v.dtype != k.dtype:
        raise RuntimeError("k and v must have the same type")
    if k.shape[0] != v.shape[0] or k.shape[1] != heads or v.shape[1] != heads:
        raise RuntimeError("k and v must have one row per token and kv head of the cache")
    if not slots.is_cuda or slots.dtype != torch.int64 or slots.dim() != 1 or slots.shape[0] != k.shape[0]:
        raise RuntimeError("slots must be an int64 CUDA tensor with one entry per token")
    dev = codes.device
    if any(t.device != dev for t in (k, v, slots)):
        raise RuntimeError("k, v, slots and the cache must be on one device")
    k, v, slots = _head_rows(k), _head_rows(v), slots.contiguous()
    with torch.cuda.device(dev):
        code = lib().uniql_kv4_append(k.data_ptr(), *_row_strides(k), v.data_ptr(), *_row_strides(v), dtype, k.shape[0], heads,
                                      k.shape[2], v.shape[2], slots.data_ptr(), codes.data_ptr(), scales.data_ptr(), pages, page, dp,
                                      status_word(dev).data_ptr(), _stream_handle(dev))
    check(code, "uniql_kv4_append")


def kv4_gather(codes: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor, cu: torch.Tensor, total: int, head_dim_k: int,
               head_dim_v: int | None = None, dtype: torch.dtype = torch.float16, starts: torch.Tensor | None = None):
    """The cached rows of a token range of every request, dequantised and packed: request i gives cu[i + 1] - cu[i] tokens from
    starts[i] on (None: from its first).  Returns k [total, kv_heads, head_dim_k] and v [total, kv_heads, head_dim_v]; places behind
    cu[-1] are zeros; tokens behind the last place are left out (status bit 2)."""
    dv = head_dim_k if head_dim_v is None else head_dim_v
    if dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("dtype must be float16 or bfloat16")
    ext = torch_ext()
    if ext is not None:
        return tuple(ext.kv4_gather(codes, scales, block_table, cu, total, head_dim_k, dv, dtype == torch.bfloat16, starts))
    pages, heads, page, dp = _cache_shape(codes, scales)
    _ints(block_table, codes, 2, "block_table")
    _ints(cu, codes, 1, "cu")
    batch = block_table.shape[0]
    if cu.shape[0] != batch + 1:
        raise RuntimeError("cu must have one entry more than block_table has rows")
    if starts is not None and _ints(starts, codes, 1, "starts").shape[0] != batch:
        raise RuntimeError("starts must have one entry per request")
    if total < 0 or head_dim_k <= 0 or dv <= 0:
        raise RuntimeError("total, head_dim_k and head_dim_v must not be negative")
    ld, dev = _ld(block_table), codes.device
    k = torch.empty(total, heads, head_dim_k, dtype=dtype, device=dev)
    v = torch.empty(total, heads, dv, dtype=dtype, device=dev)
    with torch.cuda.device(dev):
        code = lib().uniql_kv4_gather(codes.data_ptr(), scales.data_ptr(), pages, page, dp, heads, block_table.data_ptr(), ld,
                                      block_table.shape[1], batch, starts.data_ptr() if starts is not None else None, cu.data_ptr(),
                                      total, head_dim_k, dv, _DTYPE_CODE[dtype], k.data_ptr(), v.data_ptr(),
                                      status_word(dev).data_ptr(), _stream_handle(dev))
    check(code, "uniql_kv4_gather")
    return k, v


def _own_scratch(device: torch.device, nbytes: int) -> torch.Tensor:
    """Scratch of a call that a graph may replay beside eager calls and other graphs: the graph's own while the stream is captured."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(nbytes, dtype=torch.uint8, device=device)
    return _scratch_for(device, nbytes)


def kv4_attention(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                  head_dim_v: int | None = None, softmax_scale: float | None = None) -> torch.Tensor:
    """One query token per request over its first lens[i] cached tokens: q [batch, heads, channels] (fp16 or bf16), grouped heads.
    Returns [batch, heads, head_dim_v] in q's type; a request of length 0 gives zeros.  softmax_scale: 1 / sqrt(channels)."""
    if q.dim() != 3:
        raise RuntimeError("q must be a [batch, heads, channels] CUDA tensor")
    dk = q.shape[2]
    dv = dk if head_dim_v is None else head_dim_v
    scale = 1.0 / math.sqrt(max(dk, 1)) if softmax_scale is None else float(softmax_scale)
    ext = torch_ext()
    if ext is not None:
        return ext.kv4_attention(q, codes, scales, block_table, lens, dv, scale)
    pages, kv_heads, page, dp = _cache_shape(codes, scales)
    _require_cuda(q, "q")
    dtype = _kv_dtype(q, "q")
    _ints(block_table, codes, 2, "block_table")
    _ints(lens, codes, 1, "lens")
    batch, heads = q.shape[:2]
    if block_table.shape[0] != batch or lens.shape[0] != batch:
        raise RuntimeError("q, block_table and lens must have one row per request")
    if q.device != codes.device:
        raise RuntimeError("q and the cache must be on one device")
    if dv <= 0 or heads <= 0 or dk <= 0 or kv_heads <= 0 or heads % kv_heads:
        raise RuntimeError("the query heads must be a multiple of the cache's kv heads, and head sizes positive")
    ld, dev = _ld(block_table), q.device
    q = q if q.stride(2) == 1 or dk == 1 else q.contiguous()
    out = torch.empty(batch, heads, dv, dtype=q.dtype, device=dev)
    if batch == 0:
        return out
    with torch.cuda.device(dev):
        need = lib().uniql_kv4_attention_scratch_bytes(batch, heads, kv_heads, dp)
        scratch = _own_scratch(dev, need)
        code = lib().uniql_kv4_attention(q.data_ptr(), q.stride(0), q.stride(1), codes.data_ptr(), scales.data_ptr(), pages, page, dp,
                                         block_table.data_ptr(), ld, block_table.shape[1], lens.data_ptr(), batch, heads, kv_heads,
                                         dk, dv, scale, dtype, out.data_ptr(), scratch.data_ptr(), scratch.numel(),
                                         status_word(dev).data_ptr(), _stream_handle(dev))
    check(code, "uniql_kv4_attention")
    return out


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor | None = None,
                     causal: bool = True, softmax_scale: float | None = None) -> torch.Tensor:
    """Attention of packed prompts of different lengths: q [tokens, heads, channels], k and v [key tokens, kv_heads, channels] (fp16
    or bf16; views of a fused q/k/v result are fine), request i owning rows cu_q[i] .. cu_q[i + 1] - 1 of q and cu_k[i] .. of k and
    v (cu_k None: the same).  With causal the last query of a request sees all its keys, the one before it all but the last.
    Returns [tokens, heads, channels of v]; queries that see no key, and rows that no request owns, give zeros.
    A request whose rows do not all exist (cu ends behind the tensors) gives zeros, too, and raises status bit 2."""
    if q.dim() != 3:
        raise RuntimeError("q must be a [tokens, heads, channels] CUDA tensor")
    scale = 1.0 / math.sqrt(max(q.shape[2], 1)) if softmax_scale is None else float(softmax_scale)
    ext = torch_ext()
    if ext is not None:
        return ext.prompt_attention(q, k, v, cu_q, cu_k, causal, scale)
    if not (q.is_cuda and k.is_cuda and v.is_cuda) or k.dim() != 3 or v.dim() != 3:
        raise RuntimeError("q, k and v must be [tokens, heads, channels] CUDA tensors")
    dtype = _kv_dtype(q, "q")
    dev = q.device
    if k.dtype != q.dtype or v.dtype != q.dtype or k.device != dev or v.device != dev:
        raise RuntimeError("q, k and v must have the same type and device")
    if k.shape[:2] != v.shape[:2] or k.shape[2] != q.shape[2]:
        raise RuntimeError("k and v must have the same tokens and heads, q and k the same channels")
    heads, kv_heads = q.shape[1], k.shape[1]
    if heads <= 0 or kv_heads <= 0 or heads % kv_heads or q.shape[2] <= 0 or v.shape[2] <= 0:
        raise RuntimeError("the query heads must be a multiple of the kv heads, and head sizes positive")
    ck = cu_q if cu_k is None else cu_k
    _ints(cu_q, q, 1, "cu_q")
    _ints(ck, q, 1, "cu_k")
    if cu_q.shape[0] < 1 or ck.shape[0] != cu_q.shape[0]:
        raise RuntimeError("cu_q and cu_k must have one entry more than there are requests")
    q, k, v = _head_rows(q), _head_rows(k), _head_rows(v)
    out = torch.empty(q.shape[0], heads, v.shape[2], dtype=q.dtype, device=dev)
    with torch.cuda.device(dev):
        code = lib().uniql_prompt_attention(q.data_ptr(), *_row_strides(q), k.data_ptr(), *_row_strides(k), v.data_ptr(), *_row_strides(v),
                                            cu_q.data_ptr(), ck.data_ptr(), cu_q.shape[0] - 1, q.shape[0], k.shape[0], heads, kv_heads,
                                            q.shape[2], v.shape[2], scale, 1 if causal else 0, dtype, out.data_ptr(),
                                            status_word(dev).data_ptr(), _stream_handle(dev))
    check(code, "uniql_prompt_attention")
    return out
