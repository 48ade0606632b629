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


# ---------------------------------------------------------------- the int8 paged cache
# These calls take a few microseconds on the device in a decode step, so their
# checks are kept short: _here looks at a tensor once.

_current = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _here(dev, *ts):
    """Every tensor (or None) contiguous and on device `dev`."""
    for t in ts:
        if t is not None and (t.get_device() != dev or not t.is_contiguous()):
            raise ValueError(f"brain_amd.ops: tensors must be contiguous and on one GPU (device {dev}, got "
                             f"{tuple(t.shape)} on {t.get_device()}, strides {t.stride()})")


def _stream_of(dev):
    # The launches go to the current device.
    if dev < 0:
        raise ValueError("brain_amd.ops: tensors must live on the GPU")
    if dev != _current():
        raise ValueError(f"brain_amd.ops: the tensors are on GPU {dev}, the current device is {_current()}")
    return _stream()


# The C entries take sizes of 32 bits, and ctypes cuts what is longer without a
# word: sizes that could be are checked here.
_MOST, _U32 = 0x7fffffff, 0xffffffff


class PagedKV8:
    """An int8 paged KV cache (bh_kv8): pools of int32 words (4 codes each,
    n_kv * head_dim bytes a slot) and f32 scales [slots, n_kv] for keys and
    values, block_tables [batch, max_blocks] int32. Position j of sequence b is
    slot block_tables[b, j // block_size] * block_size + j % block_size. Holds
    the tensors and their addresses, so its attributes are fixed: make it once
    for a cache, and another one for other tensors (a table that has grown)."""

    def __init__(self, k_pool, v_pool, k_scales, v_scales, block_tables, block_size, head_dim):
        if head_dim <= 0 or head_dim % 4 or head_dim > 256:
            raise ValueError(f"PagedKV8: head_dim {head_dim}, a multiple of 4 up to 256")
        if not 0 < block_size <= _U32:
            raise ValueError(f"PagedKV8: block_size {block_size}")
        if k_scales.dim() != 2 or block_tables.dim() != 2:
            raise ValueError("PagedKV8: scales [slots, n_kv] and block_tables [batch, max_blocks] expected")
        slots, n_kv = k_scales.shape
        if n_kv * head_dim > _MOST or block_tables.shape[1] > _U32 or block_tables.shape[0] > _MOST // 2:
            raise ValueError(f"PagedKV8: {n_kv} kv heads, block_tables {tuple(block_tables.shape)}")
        words = slots * n_kv * head_dim // 4
        for name, t, dtype, numel in (("k_pool", k_pool, torch.int32, words), ("v_pool", v_pool, torch.int32, words),
                                      ("k_scales", k_scales, torch.float32, slots * n_kv),
                                      ("v_scales", v_scales, torch.float32, slots * n_kv),
                                      ("block_tables", block_tables, torch.int32, 0)):
            _need(t, dtype, numel, name)
        self.dev = k_pool.get_device()
        _here(self.dev, k_pool, v_pool, k_scales, v_scales, block_tables)
        self.k_pool, self.v_pool, self.k_scales, self.v_scales = k_pool, v_pool, k_scales, v_scales
        self.block_tables, self.block_size, self.head_dim, self.n_kv = block_tables, block_size, head_dim, n_kv
        self.desc = Kv8T(_ptr(k_pool), _ptr(v_pool), _ptr(k_scales), _ptr(v_scales), words, slots * n_kv,
                         _ptr(block_tables), block_tables.shape[1], block_size, n_kv, head_dim)
        self.sequences = block_tables.shape[0]
        self.needs = {}  # workspace bytes of paged_attention_i8, by the sizes of the call
        self.ref = C.byref(self.desc)

    def __setattr__(self, name, value):
        if "ref" in self.__dict__:  # (the calls read desc: a tensor put here would not reach them)
            raise AttributeError(f"PagedKV8.{name} is fixed; make another PagedKV8 for other tensors")
        super().__setattr__(name, value)


def _heads(t, dtype, hd, name):
    """(rows, heads, row stride in elements) of [rows, heads, hd] `t`, whose heads lie side by side."""
    if t.dtype != dtype:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")
    shape = t.shape
    if len(shape) != 3 or shape[2] != hd:
        raise ValueError(f"{name}: shape {tuple(shape)}, expected [rows, heads, {hd}]")
    rows, heads, _ = shape
    if rows * heads > _MOST:
        raise ValueError(f"{name}: {rows} rows of {heads} heads")
    rs, hs, es = t.stride()
    if es != 1 or (heads > 1 and hs != hd) or (rows > 1 and rs < heads * hd):
        raise ValueError(f"{name}: strides {t.stride()}; the heads of a row must lie side by side")
    return rows, heads, rs if rows > 1 else heads * hd


def _kv_batch(cache, rows, seq_lens, row_start, max_rows, max_len):
    batch = seq_lens.numel()
    _need(seq_lens, torch.int32, batch, "seq_lens")
    if batch > cache.sequences:
        raise ValueError(f"seq_lens: {batch} sequences, block_tables has {cache.sequences}")
    if row_start is None:
        if rows != batch:
            raise ValueError(f"row_start: {rows} rows of {batch} sequences need one")
    elif row_start.dtype != torch.int32 or row_start.numel() != batch + 1:
        raise ValueError(f"row_start: {row_start.numel()} entries of {row_start.dtype} for {batch} sequences")
    return Kv8BatchT(_ptr(row_start), seq_lens.data_ptr(), batch, rows, max_rows or 0, max_len or 0)


_ACT = {torch.float32: BH_OUT_F32, torch.bfloat16: BH_OUT_BF16}


def _qk_rows(dev, q, k, v, positions, inv_freq, q_weight, k_weight, eps):
    dtype = q.dtype
    if dtype not in _ACT:
        raise ValueError(f"q: dtype {dtype}, expected float32 or bfloat16")
    hd = q.shape[-1]
    if hd > 256:
        raise ValueError(f"q: head_dim {hd}, a multiple of 4 up to 256")
    rows, nh, qs = _heads(q, dtype, hd, "q")
    k_rows, nkv, ks = _heads(k, dtype, hd, "k")
    if k_rows != rows:
        raise ValueError(f"k: {k_rows} rows, q has {rows}")
    vs = 0
    if v is not None:
        vs = _heads(v, dtype, hd, "v")[2]
        if v.shape != k.shape:
            raise ValueError(f"v: shape {tuple(v.shape)}, k has {tuple(k.shape)}")
        if v.get_device() != dev:
            raise ValueError(f"v is on {v.get_device()}, q on {dev}")
    if k.get_device() != dev:
        raise ValueError(f"k is on {k.get_device()}, q on {dev}")
    _need(positions, torch.int32, rows, "positions")
    pairs = inv_freq.numel()
    _need(inv_freq, torch.float64, 0, "inv_freq")
    if 2 * pairs > hd:
        raise ValueError(f"inv_freq: {pairs} pairs, head_dim {hd}")
    if q_weight is not None:
        _need(q_weight, torch.float32, hd, "q_weight")
    if k_weight is not None:
        _need(k_weight, torch.float32, hd, "k_weight")
    _here(dev, positions, inv_freq, q_weight, k_weight)
    return QkRowsT(q.data_ptr(), k.data_ptr(), _ptr(v), qs, ks, vs, _ACT[dtype], rows, nh, nkv, hd, positions.data_ptr(),
                   inv_freq.data_ptr(), 2 * pairs, _ptr(q_weight), _ptr(k_weight), eps)


def rope_frequencies(rotary_dim, theta, device="cuda"):
    """inv_freq of plain RoPE: theta^(-2i / rotary_dim), f64 [rotary_dim / 2]."""
    return theta ** (-torch.arange(0, rotary_dim, 2, device=device, dtype=torch.float64) / rotary_dim)


def _out_like(dev, out, t, name):
    if out is None:
        out = torch.empty_like(t, memory_format=torch.contiguous_format)
        return out, out.stride(0)
    stride = _heads(out, t.dtype, t.shape[2], name)[2]
    if out.shape != t.shape or out.get_device() != dev:
        raise ValueError(f"{name}: shape {tuple(out.shape)} on {out.get_device()}, expected {tuple(t.shape)} on {dev}")
    return out, stride


def qk_norm_rope(q, k, positions, inv_freq, q_weight=None, k_weight=None, eps=1e-6, q_out=None, k_out=None):
    """Per-head RMSNorm (where a weight is given) and rotation of q [rows,
    n_heads, hd] and k [rows, n_kv, hd], f32 or bf16, views of a joined
    projection included: pair (i, i + rotary_dim/2) is turned by
    positions[row] * inv_freq[i], rotary_dim = 2 * inv_freq.numel(). Returns
    (q_out, k_out), which may be q and k themselves."""
    dev = q.get_device()
    rows = _qk_rows(dev, q, k, None, positions, inv_freq, q_weight, k_weight, eps)
    q_out, qs = _out_like(dev, q_out, q, "q_out")
    k_out, ks = _out_like(dev, k_out, k, "k_out")
    check(load().bh_qk_norm_rope(_stream_of(dev), C.byref(rows), q_out.data_ptr(), qs, k_out.data_ptr(), ks))
    return q_out, k_out


def qk_norm_rope_append_i8(q, k, v, positions, inv_freq, cache, seq_lens, row_start=None, q_weight=None, k_weight=None,
                           eps=1e-6, k_clip=None, v_clip=None, q_out=None):
    """qk_norm_rope, with the turned keys and the values quantised into the
    cache (PagedKV8): the rows row_start[b] .. row_start[b + 1] become the last
    positions of sequence b's seq_lens[b] (row_start None: one row each).
    Returns q_out."""
    dev = cache.dev
    rows = _qk_rows(dev, q, k, v, positions, inv_freq, q_weight, k_weight, eps)
    if rows.n_kv_heads != cache.n_kv or rows.head_dim != cache.head_dim:
        raise ValueError(f"k: heads {tuple(k.shape[1:])}, the cache has {(cache.n_kv, cache.head_dim)}")
    if q.get_device() != dev:
        raise ValueError(f"q is on {q.get_device()}, the cache on {dev}")
    batch = _kv_batch(cache, rows.rows, seq_lens, row_start, 0, 0)
    if k_clip is not None:
        _need(k_clip, torch.float32, cache.n_kv, "k_clip")
    if v_clip is not None:
        _need(v_clip, torch.float32, cache.n_kv, "v_clip")
    _here(dev, seq_lens, row_start, k_clip, v_clip)
    q_out, qs = _out_like(dev, q_out, q, "q_out")
    check(load().bh_qk_norm_rope_append_i8(_stream_of(dev), C.byref(rows), cache.ref, C.byref(batch), _ptr(k_clip),
                                           _ptr(v_clip), q_out.data_ptr(), qs))
    return q_out


def _queries(q, cache, seq_lens, row_start, max_rows, max_len):
    if q.dtype not in _ACT:
        raise ValueError(f"q: dtype {q.dtype}, expected float32 or bfloat16")
    rows, nh, stride = _heads(q, q.dtype, cache.head_dim, "q")
    if nh == 0 or nh % cache.n_kv:
        raise ValueError(f"q: {nh} heads over {cache.n_kv} kv heads")
    if q.get_device() != cache.dev:
        raise ValueError(f"q is on {q.get_device()}, the cache on {cache.dev}")
    batch = _kv_batch(cache, rows, seq_lens, row_start, max_rows, max_len)
    return rows, nh, stride, batch


def paged_attention_i8(q, cache, seq_lens, row_start=None, scale=None, max_rows=None, max_len=None, out=None, lse=None):
    """Causal attention of q [rows, n_heads, hd] (f32 or bf16) over the cache
    (PagedKV8): the rows row_start[b] .. row_start[b + 1] are the last of
    sequence b's seq_lens[b] positions and see the keys up to their own. scale
    defaults to hd^-0.5. max_rows and max_len, the most rows and the longest
    length where the program knows them, choose how the work is split. Returns
    (out like q, lse [rows, n_heads] f32); a row without keys has zeros and
    -inf; rows behind the last sequence stay as `out` and `lse` have them."""
    rows, nh, stride, batch = _queries(q, cache, seq_lens, row_start, max_rows, max_len)
    hd, device, dtype = cache.head_dim, q.device, q.dtype
    if out is None:
        out = q.new_empty((rows, nh, hd))
    else:
        _need(out, dtype, rows * nh * hd, "out")
    if lse is None:
        lse = torch.empty((rows, nh), device=device, dtype=torch.float32)
    else:
        _need(lse, torch.float32, rows * nh, "lse")
    _here(cache.dev, seq_lens, row_start, out, lse)
    lib, ref = load(), C.byref(batch)
    sizes = (nh, rows, batch.batch, batch.max_rows, batch.max_len, row_start is None)
    need = cache.needs.get(sizes)
    if need is None:
        n = C.c_uint64()
        check(lib.bh_paged_attention_i8_workspace(cache.ref, ref, nh, C.byref(n)))
        if len(cache.needs) > 4096:
            cache.needs.clear()
        need = cache.needs[sizes] = n.value
    ws = torch.empty(need, device=device, dtype=torch.uint8) if need else None
    check(lib.bh_paged_attention_i8(_stream_of(cache.dev), q.data_ptr(), stride, _ACT[dtype], nh, cache.ref, ref,
                                    hd ** -0.5 if scale is None else scale, out.data_ptr(), lse.data_ptr(), _ptr(ws),
                                    need))
    return out, lse


def paged_weight_sums_i8(q, lse, cache, seq_lens, acc, row_start=None, scale=None, max_rows=None, max_len=None):
    """acc [batch, n_kv, cap] f32 += the weight exp(s - lse) that the rows of
    q gave each cached key in paged_attention_i8 (same arguments, its lse),
    summed over rows and a kv head's query heads; the chunk's own keys start
    from 0. Returns acc."""
    rows, nh, stride, batch = _queries(q, cache, seq_lens, row_start, max_rows, max_len)
    _need(lse, torch.float32, rows * nh, "lse")
    if acc.dim() != 3 or acc.shape[0] < batch.batch or acc.shape[1] != cache.n_kv or acc.shape[2] > _MOST:
        raise ValueError(f"acc: shape {tuple(acc.shape)}, expected [{batch.batch}, {cache.n_kv}, cap]")
    _need(acc, torch.float32, 0, "acc")
    _here(cache.dev, seq_lens, row_start, lse, acc)
    check(load().bh_paged_weight_sums_i8(_stream_of(cache.dev), q.data_ptr(), stride, _ACT[q.dtype], nh, lse.data_ptr(),
                                         cache.ref, C.byref(batch), cache.head_dim ** -0.5 if scale is None else scale,
                                         acc.data_ptr(), acc.shape[2]))
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
    _need(seq_lens, torch.int32, batch, "seq_lens")
    _need(acc, torch.float32, 0, "acc")
    if batch > cache.sequences:
        raise ValueError(f"seq_lens: {batch} sequences, block_tables has {cache.sequences}")
    if acc.dim() != 3 or acc.shape[0] < batch or acc.shape[1] != cache.n_kv or acc.shape[2] > _MOST:
        raise ValueError(f"acc: shape {tuple(acc.shape)}, expected [{batch}, {cache.n_kv}, cap]")
    if not 0 < budget <= _MOST or sink < 0 or recent < 0 or sink + recent > budget:
        raise ValueError(f"budget {budget} with sink {sink} and recent {recent}")
    to_ptr = to_cols = out_ptr = out_cap = 0
    if out_tables is not None:
        _need(out_tables, torch.int32, 0, "out_tables")
        if out_tables.dim() != 2 or out_tables.shape[0] < batch or out_tables.shape[1] > _U32:
            raise ValueError(f"out_tables: shape {tuple(out_tables.shape)}, expected [{batch}, blocks]")
        to_ptr, to_cols = out_tables.data_ptr(), out_tables.shape[1]
    if acc_out is not None:
        _need(acc_out, torch.float32, 0, "acc_out")
        if acc_out.dim() != 3 or acc_out.shape[0] < batch or acc_out.shape[1] != cache.n_kv or acc_out.shape[2] > _U32:
            raise ValueError(f"acc_out: shape {tuple(acc_out.shape)}, expected [{batch}, {cache.n_kv}, >= {budget}]")
        out_ptr, out_cap = acc_out.data_ptr(), acc_out.shape[2]
    if keep is None:
        keep = torch.empty((batch, cache.n_kv, budget), device=acc.device, dtype=torch.int32)
    else:
        _need(keep, torch.int32, batch * cache.n_kv * budget, "keep")
    if new_lens is None:
        new_lens = torch.empty(batch, device=acc.device, dtype=torch.int32)
    else:
        _need(new_lens, torch.int32, batch, "new_lens")
    _here(cache.dev, seq_lens, acc, out_tables, acc_out, keep, new_lens)
    check(load().bh_paged_kv_evict_i8(_stream_of(cache.dev), cache.ref, seq_lens.data_ptr(), batch, acc.data_ptr(),
                                      acc.shape[2], budget, sink, recent, to_ptr, to_cols, out_ptr, out_cap,
                                      keep.data_ptr(), new_lens.data_ptr()))
    return keep, new_lens
