"""torch-tensor wrappers of the typed, stream-ordered calls in libbrain_hip.so.

torch only supplies device memory and the current HIP stream; all arithmetic
runs in the library's gfx950 kernels. Packed int8 tensors are torch.int32
tensors holding the u32 words (4 int8 per word, little-endian along K).
"""
import ctypes as C

import torch

from ._lib import BH_OUT_BF16, BH_OUT_F32, BH_OUT_I32, Kv8BatchT, Kv8T, QkRowsT, check, load

_CODES = {torch.float32: BH_OUT_F32, torch.bfloat16: BH_OUT_BF16, torch.int32: BH_OUT_I32}


# The handle of the current device's current stream. The public call builds a
# Stream object on the way (3.4 us, a third of a decode linear's host time;
# this one 0.1 us).
if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    def _stream():
        return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())
else:
    def _stream():
        return torch.cuda.current_stream().cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _dev(*ts):
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("brain_amd.ops: tensors must live on the GPU")
        if not t.is_contiguous():
            raise ValueError("brain_amd.ops: tensors must be contiguous")


def _need(t, dtype, numel, name):
    if t.dtype != dtype:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if t.numel() < numel:
        raise ValueError(f"{name}: {t.numel()} elements, needs {numel}")


def max_abs_rows(x, sx=None):
    """sx[m] = max(max|x[m,:]|, 1e-8)/127 (max_abs_row.wgsl)."""
    m, k = x.shape
    _dev(x)
    _need(x, torch.float32, m * k, "x")
    sx = torch.empty(m, device=x.device, dtype=torch.float32) if sx is None else sx
    check(load().bh_max_abs_rows(_stream(), _ptr(x), m, k, _ptr(sx)))
    return sx


def quant_pack(x, sx, xq=None):
    """xq [m, k/4] int32 words: clamp(rne(x/sx), +-127) packed (quant_pack.wgsl)."""
    m, k = x.shape
    _dev(x, sx)
    _need(x, torch.float32, m * k, "x")
    _need(sx, torch.float32, m, "sx")
    xq = torch.empty(m, k // 4, device=x.device, dtype=torch.int32) if xq is None else xq
    check(load().bh_quant_pack(_stream(), _ptr(x), _ptr(sx), m, k, _ptr(xq)))
    return xq


def quantize_rows(x, sx=None, xq=None):
    """Fused max_abs_rows + quant_pack; returns (sx, xq)."""
    m, k = x.shape
    _dev(x)
    _need(x, torch.float32, m * k, "x")
    sx = torch.empty(m, device=x.device, dtype=torch.float32) if sx is None else sx
    xq = torch.empty(m, k // 4, device=x.device, dtype=torch.int32) if xq is None else xq
    check(load().bh_quantize_rows(_stream(), _ptr(x), m, k, _ptr(sx), _ptr(xq)))
    return sx, xq


def quantize_rows_bf16(x, sx=None, xq=None):
    """Per-token quantization of bf16 activations (exactly quantize_rows of x.float())."""
    m, k = x.shape
    _dev(x)
    _need(x, torch.bfloat16, m * k, "x")
    sx = torch.empty(m, device=x.device, dtype=torch.float32) if sx is None else sx
    xq = torch.empty(m, k // 4, device=x.device, dtype=torch.int32) if xq is None else xq
    check(load().bh_quantize_rows_bf16(_stream(), _ptr(x), m, k, _ptr(sx), _ptr(xq)))
    return sx, xq


_VARIANTS = {"auto": "bh_matmul_i8", "gemv": "bh_matmul_i8_gemv", "dyn": "bh_matmul_i8_dyn"}


def matmul_i8(xq, wq, sx, sw, bias=None, out_dtype=torch.float32, variant="auto", out=None):
    """out[m,n] = (f32(xq.wq^T) * sx[m]) * sw[n] (+ bias[n]), f32 or bf16;
    out_dtype=torch.int32 returns the raw i32 accumulators."""
    m, kg = xq.shape
    n = wq.shape[0]
    _dev(xq, wq, sx, sw, bias, out)
    _need(xq, torch.int32, m * kg, "xq")
    _need(wq, torch.int32, n * kg, "wq")
    _need(sx, torch.float32, m, "sx")
    _need(sw, torch.float32, n, "sw")
    if bias is not None:
        _need(bias, torch.float32, n, "bias")
    code = _CODES[out_dtype]
    out = torch.empty(m, n, device=xq.device, dtype=out_dtype) if out is None else out
    _need(out, out_dtype, m * n, "out")
    fn = getattr(load(), _VARIANTS[variant])
    check(fn(_stream(), _ptr(xq), _ptr(wq), _ptr(sx), _ptr(sw), _ptr(bias), _ptr(out), code, m, kg, n))
    return out


def matmul_i8_quant(xq, wq, sx, sw, bias=None, out=None, sx_out=None, xq_out=None):
    """bf16 out[m,n] = matmul_i8_dyn(xq, wq, sx, sw, bias), then the per-row
    quantization of out (quantize_rows_bf16) into sx_out [m], xq_out [m, n/4]
    for the next linear, in one call (split-K GEMMs reduce and quantize in one
    pass). sx_out may be sx and xq_out may overlap xq."""
    m, kg = xq.shape
    n = wq.shape[0]
    if n % 4:
        raise ValueError(f"matmul_i8_quant: n={n} is not a multiple of 4")
    _dev(xq, wq, sx, sw, bias, out, sx_out, xq_out)
    _need(xq, torch.int32, m * kg, "xq")
    _need(wq, torch.int32, n * kg, "wq")
    _need(sx, torch.float32, m, "sx")
    _need(sw, torch.float32, n, "sw")
    if bias is not None:
        _need(bias, torch.float32, n, "bias")
    out = torch.empty(m, n, device=xq.device, dtype=torch.bfloat16) if out is None else out
    sx_out = torch.empty(m, device=xq.device, dtype=torch.float32) if sx_out is None else sx_out
    xq_out = torch.empty(m, n // 4, device=xq.device, dtype=torch.int32) if xq_out is None else xq_out
    _need(out, torch.bfloat16, m * n, "out")
    _need(sx_out, torch.float32, m, "sx_out")
    _need(xq_out, torch.int32, m * n // 4, "xq_out")
    check(load().bh_matmul_i8_dyn_quant(_stream(), _ptr(xq), _ptr(wq), _ptr(sx), _ptr(sw), _ptr(bias), _ptr(out),
                                        m, kg, n, _ptr(sx_out), _ptr(xq_out)))
    return out, sx_out, xq_out


def matmul_i8_static(xq, wq, sx, sw, out=None):
    """matmul_i8.wgsl: out = f32(acc) * (sx*sw) with scalar per-tensor scales."""
    m, kg = xq.shape
    n = wq.shape[0]
    _dev(xq, wq, out)
    _need(xq, torch.int32, m * kg, "xq")
    _need(wq, torch.int32, n * kg, "wq")
    out = torch.empty(m, n, device=xq.device, dtype=torch.float32) if out is None else out
    _need(out, torch.float32, m * n, "out")
    check(load().bh_matmul_i8_static(_stream(), _ptr(xq), _ptr(wq), float(sx), float(sw), _ptr(out), m, kg, n))
    return out


def linear_i8(x, wq, sw, bias=None, out_dtype=torch.float32, sx=None, xq=None, out=None):
    """Quantize x per token, then the W8A8 matmul (Ops::act + Ops::matmul)."""
    m, k = x.shape
    n = wq.shape[0]
    if k % 4:
        raise ValueError(f"linear_i8: k={k} is not a multiple of 4")
    _dev(x, wq, sw, bias, sx, xq, out)
    _need(x, torch.float32, m * k, "x")
    _need(wq, torch.int32, n * (k // 4), "wq")
    _need(sw, torch.float32, n, "sw")
    if bias is not None:
        _need(bias, torch.float32, n, "bias")
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"linear_i8: out_dtype {out_dtype}, expected float32 or bfloat16")
    if sx is None and xq is None:  # one allocation for both: [m, k/4] codes, then [m] scales
        scratch = torch.empty(m * (k // 4) + m, device=x.device, dtype=torch.int32)
        xq_ptr = scratch.data_ptr()
        sx_ptr = xq_ptr + m * k
    else:
        sx = torch.empty(m, device=x.device, dtype=torch.float32) if sx is None else sx
        xq = torch.empty(m, k // 4, device=x.device, dtype=torch.int32) if xq is None else xq
        _need(sx, torch.float32, m, "sx")
        _need(xq, torch.int32, m * (k // 4), "xq")
        sx_ptr, xq_ptr = sx.data_ptr(), xq.data_ptr()
    code = BH_OUT_F32 if out_dtype == torch.float32 else BH_OUT_BF16
    out = torch.empty(m, n, device=x.device, dtype=out_dtype) if out is None else out
    _need(out, out_dtype, m * n, "out")
    check(load().bh_linear_i8(_stream(), _ptr(x), _ptr(wq), _ptr(sw), _ptr(bias), sx_ptr, xq_ptr, _ptr(out), code, m, k,
                              n))
    return out


def quantize_weight_device(w):
    """Per-output-channel weight quantization on the GPU (int8.rs quantize_weight)."""
    n, k = w.shape
    _dev(w)
    packed = torch.empty(n, k // 4, device=w.device, dtype=torch.int32)
    sw = torch.empty(n, device=w.device, dtype=torch.float32)
    check(load().bh_quantize_weight_device(_stream(), _ptr(w), n, k, _ptr(packed), _ptr(sw)))
    return packed, sw


def f32_to_bf16(x):
    """bf16 bit patterns (int16 tensor) of f32 `x`, the library's output rounding (half.rs f32_to_bf16)."""
    _dev(x)
    out = torch.empty(x.shape, device=x.device, dtype=torch.int16)
    check(load().bh_f32_to_bf16(_stream(), _ptr(x), _ptr(out), x.numel()))
    return out


def reserve_workspace(m, k, n, stream=None):
    """Pre-size the workspaces of `stream` (default: current) that an
    [m,k] x [n,k] GEMM may take (split-K slabs; from 6144 rows the int8
    expansion of int4 weights); required before capturing a GEMM that splits K
    in a graph, which must then not run concurrently with other work that uses
    the stream's workspaces."""
    sp = (stream or torch.cuda.current_stream()).cuda_stream
    check(load().bh_reserve_workspace(sp, m, k // 4, n))


_Q4_VARIANTS = {"auto": "bh_matmul_q4", "gemv": "bh_matmul_q4_gemv", "dyn": "bh_matmul_q4_dyn"}


def matmul_q4(xq, wq4, sx, sw, bias=None, out_dtype=torch.float32, variant="auto", out=None):
    """W4A8: xq [m, k/4] int8 activation words, wq4 [n, k/8] int4 weight words
    (crates/model/src/int4.rs), (f32(acc)*sx)*sw (+bias) -> out [m, n]."""
    m, kg = xq.shape
    n, kw = wq4.shape
    k = kg * 4
    if kw * 8 != k:
        raise ValueError(f"matmul_q4: xq has K={k}, wq4 has K={kw * 8}")
    _dev(xq, wq4, sx, sw, bias, out)
    _need(xq, torch.int32, m * kg, "xq")
    _need(wq4, torch.int32, n * kw, "wq4")
    _need(sx, torch.float32, m, "sx")
    _need(sw, torch.float32, n, "sw")
    if bias is not None:
        _need(bias, torch.float32, n, "bias")
    code = _CODES[out_dtype]
    out = torch.empty(m, n, device=xq.device, dtype=out_dtype) if out is None else out
    _need(out, out_dtype, m * n, "out")
    check(getattr(load(), _Q4_VARIANTS[variant])(
        _stream(), _ptr(xq), _ptr(wq4), _ptr(sx), _ptr(sw), _ptr(bias), _ptr(out), code, m, k, n))
    return out


def moe_linear_gated_i8(xq, wq, sx, sw, gate, e_idx, out=None):
    """moe_linear_gated_i8.wgsl: f32 out [m, n], rows with gate[row, e_idx] <= 0 are +0."""
    m, kg = xq.shape
    n = wq.shape[0]
    n_experts = gate.shape[1]
    _dev(xq, wq, sx, sw, gate, out)
    _need(xq, torch.int32, m * kg, "xq")
    _need(wq, torch.int32, n * kg, "wq")
    _need(sx, torch.float32, m, "sx")
    _need(sw, torch.float32, n, "sw")
    _need(gate, torch.float32, m * n_experts, "gate")
    out = torch.empty(m, n, device=xq.device, dtype=torch.float32) if out is None else out
    _need(out, torch.float32, m * n, "out")
    check(load().bh_moe_linear_gated_i8(_stream(), _ptr(xq), _ptr(wq), _ptr(sx), _ptr(sw), _ptr(gate), n_experts,
                                        e_idx, _ptr(out), m, kg, n))
    return out


class PagedKV8:
    """An int8 paged KV cache (bh_kv8): pools of int32 words (4 codes each,
    n_kv * head_dim bytes a slot) and f32 scales [slots, n_kv] for keys and
    values, block_tables [batch, max_blocks] int32. Position j of sequence b is
    slot block_tables[b, j // block_size] * block_size + j % block_size. Holds
    the tensors; make it once for a cache."""

    def __init__(self, k_pool, v_pool, k_scales, v_scales, block_tables, block_size, head_dim):
        _dev(k_pool, v_pool, k_scales, v_scales, block_tables)
        if head_dim <= 0 or head_dim % 4 or head_dim > 256:
            raise ValueError(f"PagedKV8: head_dim {head_dim}, a multiple of 4 up to 256")
        if block_size <= 0:
            raise ValueError(f"PagedKV8: block_size {block_size}")
        if k_scales.dim() != 2 or block_tables.dim() != 2:
            raise ValueError("PagedKV8: scales [slots, n_kv] and block_tables [batch, max_blocks] expected")
        slots, n_kv = k_scales.shape
        for name, t, dtype, numel in (("k_pool", k_pool, torch.int32, slots * n_kv * head_dim // 4),
                                      ("v_pool", v_pool, torch.int32, slots * n_kv * head_dim // 4),
                                      ("k_scales", k_scales, torch.float32, slots * n_kv),
                                      ("v_scales", v_scales, torch.float32, slots * n_kv),
                                      ("block_tables", block_tables, torch.int32, 0)):
            _need(t, dtype, numel, name)
            if t.device != k_pool.device:
                raise ValueError(f"PagedKV8: {name} is on {t.device}, k_pool on {k_pool.device}")
        self.k_pool, self.v_pool, self.k_scales, self.v_scales = k_pool, v_pool, k_scales, v_scales
        self.block_tables, self.block_size, self.head_dim, self.n_kv = block_tables, block_size, head_dim, n_kv
        self.device = k_pool.device
        self.desc = Kv8T(_ptr(k_pool), _ptr(v_pool), _ptr(k_scales), _ptr(v_scales), slots * n_kv * head_dim // 4,
                         slots * n_kv, _ptr(block_tables), block_tables.shape[1], block_size, n_kv, head_dim)


def _heads(t, dtype, hd, name):
    """Row stride (elements) of [rows, heads, hd] `t`, whose heads lie side by side."""
    if t.dtype != dtype:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if not t.is_cuda:
        raise ValueError("brain_amd.ops: tensors must live on the GPU")
    if t.dim() != 3 or t.shape[2] != hd:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected [rows, heads, {hd}]")
    rs, hs, es = t.stride()
    rows, heads = t.shape[0], t.shape[1]
    if (hd > 1 and es != 1) or (heads > 1 and hs != hd) or (rows > 1 and rs < heads * hd):
        raise ValueError(f"{name}: strides {t.stride()}; the heads of a row must lie side by side")
    return rs if rows > 1 else heads * hd


def _same_device(device, **ts):
    # The launches go to the current device's current stream.
    if device.index is not None and device.index != torch.cuda.current_device():
        raise ValueError(f"brain_amd.ops: the tensors are on {device}, the current device is "
                         f"{torch.cuda.current_device()}")
    for name, t in ts.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, expected {device}")


def _kv_batch(cache, rows, seq_lens, row_start, max_rows, max_len):
    batch = seq_lens.numel()
    _dev(seq_lens, row_start)
    _need(seq_lens, torch.int32, batch, "seq_lens")
    if batch > cache.block_tables.shape[0]:
        raise ValueError(f"seq_lens: {batch} sequences, block_tables has {cache.block_tables.shape[0]}")
    if row_start is None:
        if rows != batch:
            raise ValueError(f"row_start: {rows} rows of {batch} sequences need one")
    else:
        _need(row_start, torch.int32, batch + 1, "row_start")
        if row_start.numel() != batch + 1:
            raise ValueError(f"row_start: {row_start.numel()} entries for {batch} sequences")
    return Kv8BatchT(_ptr(row_start), _ptr(seq_lens), batch, rows, max_rows or 0, max_len or 0)


_ACT = {torch.float32: BH_OUT_F32, torch.bfloat16: BH_OUT_BF16}


def _qk_rows(q, k, v, positions, inv_freq, q_weight, k_weight, eps):
    if q.dtype not in _ACT:
        raise ValueError(f"q: dtype {q.dtype}, expected float32 or bfloat16")
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q, k: [rows, heads, head_dim] expected")
    rows, nh, hd = q.shape
    nkv = k.shape[1]
    strides = [_heads(q, q.dtype, hd, "q"), _heads(k, q.dtype, hd, "k"), 0]
    if k.shape[0] != rows:
        raise ValueError(f"k: {k.shape[0]} rows, q has {rows}")
    if v is not None:
        strides[2] = _heads(v, q.dtype, hd, "v")
        if v.shape != k.shape:
            raise ValueError(f"v: shape {tuple(v.shape)}, k has {tuple(k.shape)}")
    _dev(positions, inv_freq, q_weight, k_weight)
    _need(positions, torch.int32, rows, "positions")
    _need(inv_freq, torch.float64, 0, "inv_freq")
    if 2 * inv_freq.numel() > hd:
        raise ValueError(f"inv_freq: {inv_freq.numel()} pairs, head_dim {hd}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            _need(w, torch.float32, hd, name)
    _same_device(q.device, k=k, v=v, positions=positions, inv_freq=inv_freq, q_weight=q_weight, k_weight=k_weight)
    return QkRowsT(q.data_ptr(), k.data_ptr(), _ptr(v), *strides, _ACT[q.dtype], rows, nh, nkv, hd, _ptr(positions),
                   _ptr(inv_freq), 2 * inv_freq.numel(), _ptr(q_weight), _ptr(k_weight), eps)


def rope_frequencies(rotary_dim, theta, device="cuda"):
    """inv_freq of plain RoPE: theta^(-2i / rotary_dim), f64 [rotary_dim / 2]."""
    return theta ** (-torch.arange(0, rotary_dim, 2, device=device, dtype=torch.float64) / rotary_dim)


def _out_like(out, t, name):
    if out is None:
        return torch.empty(t.shape, device=t.device, dtype=t.dtype), t.shape[1] * t.shape[2]
    stride = _heads(out, t.dtype, t.shape[2], name)
    if out.shape != t.shape:
        raise ValueError(f"{name}: shape {tuple(out.shape)}, expected {tuple(t.shape)}")
    _same_device(t.device, **{name: out})
    return out, stride


def qk_norm_rope(q, k, positions, inv_freq, q_weight=None, k_weight=None, eps=1e-6, q_out=None, k_out=None):
    """Per-head RMSNorm (where a weight is given) and rotation of q [rows,
    n_heads, hd] and k [rows, n_kv, hd], f32 or bf16, views of a joined
    projection included: pair (i, i + rotary_dim/2) is turned by
    positions[row] * inv_freq[i], rotary_dim = 2 * inv_freq.numel(). Returns
    (q_out, k_out), which may be q and k themselves."""
    rows = _qk_rows(q, k, None, positions, inv_freq, q_weight, k_weight, eps)
    q_out, qs = _out_like(q_out, q, "q_out")
    k_out, ks = _out_like(k_out, k, "k_out")
    check(load().bh_qk_norm_rope(_stream(), C.byref(rows), q_out.data_ptr(), qs, k_out.data_ptr(), ks))
    return q_out, k_out


def qk_norm_rope_append_i8(q, k, v, positions, inv_freq, cache, seq_lens, row_start=None, q_weight=None, k_weight=None,
                           eps=1e-6, k_clip=None, v_clip=None, q_out=None):
    """qk_norm_rope, with the turned keys and the values quantised into the
    cache (PagedKV8): the rows row_start[b] .. row_start[b + 1] become the last
    positions of sequence b's seq_lens[b] (row_start None: one row each).
    Returns q_out."""
    rows = _qk_rows(q, k, v, positions, inv_freq, q_weight, k_weight, eps)
    if (k.shape[1], k.shape[2]) != (cache.n_kv, cache.head_dim):
        raise ValueError(f"k: heads {tuple(k.shape[1:])}, the cache has {(cache.n_kv, cache.head_dim)}")
    batch = _kv_batch(cache, q.shape[0], seq_lens, row_start, 0, 0)
    _dev(k_clip, v_clip)
    for name, t in (("k_clip", k_clip), ("v_clip", v_clip)):
        if t is not None:
            _need(t, torch.float32, cache.n_kv, name)
    _same_device(q.device, cache=cache, seq_lens=seq_lens, row_start=row_start, k_clip=k_clip, v_clip=v_clip)
    q_out, qs = _out_like(q_out, q, "q_out")
    check(load().bh_qk_norm_rope_append_i8(_stream(), C.byref(rows), C.byref(cache.desc), C.byref(batch), _ptr(k_clip),
                                           _ptr(v_clip), q_out.data_ptr(), qs))
    return q_out


def _queries(q, cache, seq_lens, row_start, max_rows, max_len):
    if q.dtype not in _ACT:
        raise ValueError(f"q: dtype {q.dtype}, expected float32 or bfloat16")
    stride = _heads(q, q.dtype, cache.head_dim, "q")
    if q.shape[1] == 0 or q.shape[1] % cache.n_kv:
        raise ValueError(f"q: {q.shape[1]} heads over {cache.n_kv} kv heads")
    batch = _kv_batch(cache, q.shape[0], seq_lens, row_start, max_rows, max_len)
    _same_device(q.device, cache=cache, seq_lens=seq_lens, row_start=row_start)
    return stride, batch


def paged_attention_i8(q, cache, seq_lens, row_start=None, scale=None, max_rows=None, max_len=None, out=None, lse=None):
    """Causal attention of q [rows, n_heads, hd] (f32 or bf16) over the cache
    (PagedKV8): the rows row_start[b] .. row_start[b + 1] are the last of
    sequence b's seq_lens[b] positions and see the keys up to their own. scale
    defaults to hd^-0.5. max_rows and max_len, the most rows and the longest
    length where the program knows them, choose how the work is split. Returns
    (out like q, lse [rows, n_heads] f32); a row without keys has zeros and
    -inf; rows behind the last sequence stay as `out` and `lse` have them."""
    stride, batch = _queries(q, cache, seq_lens, row_start, max_rows, max_len)
    rows, nh, hd = q.shape
    if out is None:
        out = torch.empty(rows, nh, hd, device=q.device, dtype=q.dtype)
    if lse is None:
        lse = torch.empty(rows, nh, device=q.device, dtype=torch.float32)
    _dev(out, lse)
    _need(out, q.dtype, rows * nh * hd, "out")
    _need(lse, torch.float32, rows * nh, "lse")
    _same_device(q.device, out=out, lse=lse)
    lib, need = load(), C.c_uint64()
    check(lib.bh_paged_attention_i8_workspace(C.byref(cache.desc), C.byref(batch), nh, C.byref(need)))
    ws = torch.empty(need.value, device=q.device, dtype=torch.uint8) if need.value else None
    check(lib.bh_paged_attention_i8(_stream(), q.data_ptr(), stride, _ACT[q.dtype], nh, C.byref(cache.desc),
                                    C.byref(batch), hd ** -0.5 if scale is None else scale, out.data_ptr(),
                                    lse.data_ptr(), _ptr(ws), need.value))
    return out, lse


def paged_weight_sums_i8(q, lse, cache, seq_lens, acc, row_start=None, scale=None, max_rows=None, max_len=None):
    """acc [batch, n_kv, cap] f32 += the weight exp(s - lse) that the rows of
    q gave each cached key in paged_attention_i8 (same arguments, its lse),
    summed over rows and a kv head's query heads; the chunk's own keys start
    from 0. Returns acc."""
    stride, batch = _queries(q, cache, seq_lens, row_start, max_rows, max_len)
    rows, nh, hd = q.shape
    _dev(lse, acc)
    _need(lse, torch.float32, rows * nh, "lse")
    if acc.dim() != 3 or acc.shape[0] < seq_lens.numel() or acc.shape[1] != cache.n_kv:
        raise ValueError(f"acc: shape {tuple(acc.shape)}, expected [{seq_lens.numel()}, {cache.n_kv}, cap]")
    _need(acc, torch.float32, 0, "acc")
    _same_device(q.device, lse=lse, acc=acc)
    check(load().bh_paged_weight_sums_i8(_stream(), q.data_ptr(), stride, _ACT[q.dtype], nh, _ptr(lse),
                                         C.byref(cache.desc), C.byref(batch), hd ** -0.5 if scale is None else scale,
                                         _ptr(acc), acc.shape[2]))
    return acc


def paged_kv_evict_i8(cache, seq_lens, acc, budget, sink=0, recent=0, out_tables=None, acc_out=None, keep=None,
                      new_lens=None):
    """Cut sequences longer than `budget` down to it: each kv head keeps its
    first `sink` positions, its last `recent` and the heaviest between by acc
    [batch, n_kv, cap] (ties: the lower position). The entries kept move, in
    order, to the front of the sequence: of out_tables' blocks [batch, blocks],
    or, without, of its own. acc_out [batch, n_kv, >= budget] takes their acc
    (it may be acc). Returns (keep [batch, n_kv, budget] int32, -1 behind the
    last one, new_lens [batch])."""
    batch = seq_lens.numel()
    _dev(seq_lens, acc, out_tables, acc_out, keep, new_lens)
    _need(seq_lens, torch.int32, batch, "seq_lens")
    _need(acc, torch.float32, 0, "acc")
    if batch > cache.block_tables.shape[0]:
        raise ValueError(f"seq_lens: {batch} sequences, block_tables has {cache.block_tables.shape[0]}")
    if acc.dim() != 3 or acc.shape[0] < batch or acc.shape[1] != cache.n_kv:
        raise ValueError(f"acc: shape {tuple(acc.shape)}, expected [{batch}, {cache.n_kv}, cap]")
    if budget <= 0 or sink < 0 or recent < 0 or sink + recent > budget:
        raise ValueError(f"budget {budget} with sink {sink} and recent {recent}")
    if out_tables is not None:
        _need(out_tables, torch.int32, 0, "out_tables")
        if out_tables.dim() != 2 or out_tables.shape[0] < batch:
            raise ValueError(f"out_tables: shape {tuple(out_tables.shape)}, expected [{batch}, blocks]")
    if acc_out is not None:
        _need(acc_out, torch.float32, 0, "acc_out")
        if acc_out.dim() != 3 or acc_out.shape[0] < batch or acc_out.shape[1] != cache.n_kv:
            raise ValueError(f"acc_out: shape {tuple(acc_out.shape)}, expected [{batch}, {cache.n_kv}, >= {budget}]")
    keep = torch.empty(batch, cache.n_kv, budget, device=acc.device, dtype=torch.int32) if keep is None else keep
    new_lens = torch.empty(batch, device=acc.device, dtype=torch.int32) if new_lens is None else new_lens
    _need(keep, torch.int32, batch * cache.n_kv * budget, "keep")
    _need(new_lens, torch.int32, batch, "new_lens")
    _same_device(cache.device, seq_lens=seq_lens, acc=acc, out_tables=out_tables, acc_out=acc_out, keep=keep,
                 new_lens=new_lens)
    check(load().bh_paged_kv_evict_i8(_stream(), C.byref(cache.desc), _ptr(seq_lens), batch, _ptr(acc), acc.shape[2],
                                      budget, sink, recent, _ptr(out_tables),
                                      out_tables.shape[1] if out_tables is not None else 0, _ptr(acc_out),
                                      acc_out.shape[2] if acc_out is not None else 0, _ptr(keep), _ptr(new_lens)))
    return keep, new_lens
