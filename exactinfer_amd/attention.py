"""Torch-tensor front end of the gfx950 attention path (calls the C ABI, nothing else).

Each function launches on torch's current HIP stream and validates shapes on the host
before any launch (the C ABI validates again).  Tensors are float32, contiguous in the
innermost dimension, on the GPU.

The names follow the reference's per-layer attention steps (src/cuda/model_cuda.cu:
1797-1822): headnorm_rope -> kv_append -> attn_decode (B == 1) or attn_prefill (B > 1).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _capi

HEAD_DIM = 128


def _stream() -> int:
    # the raw handle of torch's current stream: torch.cuda.current_stream() builds a Stream object around it
    # (2.6 us against 0.25 us, every call; a decode step's two launches take 7.2 us)
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _stream_on(dev: int) -> int:
    return torch._C._cuda_getCurrentRawStream(dev)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _need_gpu_f32(name: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    if t.dtype != torch.float32:
        raise ValueError(f"{name} must be float32, got {t.dtype}")
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")


def _scale_of(head_dim: float) -> float:
    one, d = torch.tensor((1.0, head_dim), dtype=torch.float32, device="cpu")
    return float(one / torch.sqrt(d))


_SCALE = _scale_of(float(HEAD_DIM))  # made once: as tensor operations it takes 4 us, in every call


def default_scale(head_dim: int = HEAD_DIM) -> float:
    """1/sqrt(D) rounded to float as the reference does (src/model.cpp:163, src/cuda/model_cuda.cu:1786)."""
    return _SCALE if head_dim is HEAD_DIM else _scale_of(float(head_dim))


@dataclass(frozen=True)
class AttnShape:
    """The Config fields the path reads (src/model.h:17-23)."""

    n_head: int
    n_head_kv: int
    head_dim: int = HEAD_DIM
    rope_dim: int = HEAD_DIM
    rope_base: float = 1e6
    eps: float = 1e-6

    @property
    def group(self) -> int:
        return self.n_head // self.n_head_kv

    @property
    def kd(self) -> int:
        return self.n_head_kv * self.head_dim

    @property
    def qkv(self) -> int:
        return (self.n_head + 2 * self.n_head_kv) * self.head_dim


# ---------------------------------------------------------------- RoPE table
def rope_table(n_ctx: int, rope_dim: int = HEAD_DIM, theta: float = 1e6, device="cuda") -> torch.Tensor:
    """[n_ctx, rope_dim/2, 2] (cos, sin) float table, angles in double (src/cuda/model_cuda.cu:1610-1619)."""
    host = torch.empty((n_ctx, rope_dim // 2, 2), dtype=torch.float32)
    _capi.call("ei_rope_table_fill", host.data_ptr(), n_ctx, rope_dim, float(theta))
    return host.to(device) if device != "cpu" else host


# ---------------------------------------------------------------- prologue
def headnorm_rope(buf: torch.Tensor, n_heads: int, gamma: torch.Tensor, cs: torch.Tensor, pos_dev: torch.Tensor,
                  rope_dim: int = HEAD_DIM, eps: float = 1e-6, rows: int | None = None) -> None:
    """In place on buf[rows, row_stride] (heads at column h*128)."""
    _need_gpu_f32("buf", buf)
    rows = buf.shape[0] if rows is None else rows
    _capi.call("ei_headnorm_rope", _stream(), buf.data_ptr(), rows, buf.stride(0), n_heads, HEAD_DIM,
               gamma.data_ptr(), cs.data_ptr(), pos_dev.data_ptr(), rope_dim, float(eps))


def kv_append(k_src: torch.Tensor, v_src: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor,
              pos_dev: torch.Tensor) -> None:
    """Copy rows of k_src/v_src ([rows, >=kd], same row stride) into cache rows *pos_dev + b."""
    for n, t in (("k_src", k_src), ("v_src", v_src), ("kc", kc), ("vc", vc)):
        _need_gpu_f32(n, t)
    if k_src.stride(0) != v_src.stride(0):
        raise ValueError("k_src and v_src must share a row stride")
    kd = kc.shape[-1] * (kc.shape[-2] if kc.dim() == 3 else 1)
    _capi.call("ei_kv_append", _stream(), k_src.data_ptr(), v_src.data_ptr(), k_src.stride(0), k_src.shape[0],
               kc.data_ptr(), vc.data_ptr(), kd, pos_dev.data_ptr())


def qkv_prepare(qkv: torch.Tensor, shape: AttnShape, q_gamma: torch.Tensor, k_gamma: torch.Tensor,
                cs: torch.Tensor, pos_dev: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor) -> None:
    """Fused QK-norm + RoPE (in place) and K/V append for a [rows, (H+2HKV)*128] buffer."""
    _need_gpu_f32("qkv", qkv)
    _capi.call("ei_qkv_prepare", _stream(), qkv.data_ptr(), qkv.shape[0], qkv.stride(0), shape.n_head,
               shape.n_head_kv, shape.head_dim, q_gamma.data_ptr(), k_gamma.data_ptr(), cs.data_ptr(),
               pos_dev.data_ptr(), shape.rope_dim, float(shape.eps), kc.data_ptr(), vc.data_ptr())


# ---------------------------------------------------------------- decode
class DecodeWorkspace:
    """Split-K partials + arrival counters, sized for (n_seq, max_kv); cleared once here."""

    def __init__(self, n_seq: int, n_head: int, n_head_kv: int, max_kv: int, device="cuda"):
        self.n_seq, self.max_kv = n_seq, max_kv
        self.nbytes = int(_capi.lib().ei_attn_decode_ws_bytes(n_seq, n_head, n_head_kv, max_kv))
        if self.nbytes == 0:
            raise ValueError("invalid decode workspace shape")
        self.buf = torch.empty(self.nbytes, dtype=torch.uint8, device=device)
        _capi.call("ei_attn_workspace_init", _stream(), self.buf.data_ptr(), self.nbytes)

    def status(self) -> int:
        """The workspace's sticky status word (uint32 at (nbytes - 256) & ~255; bit 0: the splits of one
        (sequence, KV head) ran on different XCDs, against the placement the in-kernel split
        merge relies on).  Read through ei_attn_workspace_status, which synchronises the stream."""
        import ctypes
        word = ctypes.c_uint32(0)
        _capi.call("ei_attn_workspace_status", _stream(), self.buf.data_ptr(), self.nbytes, ctypes.byref(word))
        return int(word.value)

    def check(self) -> None:
        """Raises EiError (EI_ERR_MERGE) when the status word reports a failed split-merge check."""
        _capi.call("ei_decode_status_check", self.status())


def attn_decode(q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, pos_dev: torch.Tensor, shape: AttnShape,
                ws: DecodeWorkspace, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """q [H, 128] (normed + roped); keys 0..*pos_dev of the [n_ctx, HKV, 128] cache; returns [H, 128]."""
    _need_gpu_f32("q", q)
    out = torch.empty((shape.n_head, HEAD_DIM), dtype=torch.float32, device=q.device) if out is None else out
    scale = default_scale() if scale is None else scale
    _capi.call("ei_attn_decode", _stream(), q.data_ptr(), out.data_ptr(), kc.data_ptr(), vc.data_ptr(),
               pos_dev.data_ptr(), shape.n_head, shape.n_head_kv, shape.head_dim, float(scale), ws.max_kv,
               ws.buf.data_ptr(), ws.nbytes)
    return out


def attn_decode_batched(q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, kv_offset: torch.Tensor,
                        kv_len: torch.Tensor, shape: AttnShape, ws: DecodeWorkspace, scale: float | None = None,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """q [n_seq, H*128 (or wider rows)]; kv_offset int64 / kv_len int32 device arrays; returns [n_seq, H, 128]."""
    n_seq = kv_len.shape[0]
    out = torch.empty((n_seq, shape.n_head, HEAD_DIM), dtype=torch.float32, device=q.device) if out is None else out
    scale = default_scale() if scale is None else scale
    if kv_offset.dtype != torch.int64 or kv_len.dtype != torch.int32:
        raise ValueError("kv_offset must be int64 and kv_len int32")
    _capi.call("ei_attn_decode_batched", _stream(), q.data_ptr(), q.stride(0), out.data_ptr(), kc.data_ptr(),
               vc.data_ptr(), kv_offset.data_ptr(), kv_len.data_ptr(), n_seq, shape.n_head, shape.n_head_kv,
               shape.head_dim, float(scale), ws.max_kv, ws.buf.data_ptr(), ws.nbytes)
    return out


def decode_step(qkv: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, shape: AttnShape, q_gamma: torch.Tensor,
                k_gamma: torch.Tensor, cs: torch.Tensor, ws: DecodeWorkspace, pos_dev: torch.Tensor | None = None,
                kv_offset: torch.Tensor | None = None, kv_len: torch.Tensor | None = None,
                scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Fused one-token step: norm+RoPE, KV append, attention.  qkv [n_seq, (H+2HKV)*128]."""
    _need_gpu_f32("qkv", qkv)
    n_seq = qkv.shape[0] if qkv.dim() == 2 else 1
    out = torch.empty((n_seq, shape.n_head, HEAD_DIM), dtype=torch.float32, device=qkv.device) if out is None else out
    scale = default_scale() if scale is None else scale
    _capi.call("ei_decode_step", _stream(), qkv.data_ptr(), qkv.stride(0) if qkv.dim() == 2 else shape.qkv,
               out.data_ptr(), kc.data_ptr(), vc.data_ptr(), _ptr(kv_offset), _ptr(kv_len), _ptr(pos_dev), n_seq,
               shape.n_head, shape.n_head_kv, shape.head_dim, q_gamma.data_ptr(), k_gamma.data_ptr(),
               cs.data_ptr(), shape.rope_dim, float(shape.eps), float(scale), ws.max_kv, ws.buf.data_ptr(),
               ws.nbytes)
    return out


def attn_decode_paged(q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, block_table: torch.Tensor,
                      block_size: int, kv_len: torch.Tensor, shape: AttnShape, ws: DecodeWorkspace,
                      scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Paged multi-sequence decode: block_table int32 [n_seq, max_blocks] of physical blocks of
    `block_size` rows in the pool kc/vc; q [n_seq, >= H*128]; returns [n_seq, H, 128]."""
    _need_gpu_f32("q", q)
    n_seq, max_blocks = block_table.shape
    out = torch.empty((n_seq, shape.n_head, HEAD_DIM), dtype=torch.float32, device=q.device) if out is None else out
    scale = default_scale() if scale is None else scale
    _capi.call("ei_attn_decode_paged", _stream(), q.data_ptr(), q.stride(0), out.data_ptr(), kc.data_ptr(),
               vc.data_ptr(), block_table.data_ptr(), max_blocks, block_size, kv_len.data_ptr(), n_seq, shape.n_head,
               shape.n_head_kv, shape.head_dim, float(scale), ws.max_kv, ws.buf.data_ptr(), ws.nbytes)
    return out


def decode_step_paged(qkv: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, block_table: torch.Tensor,
                      block_size: int, kv_len: torch.Tensor, shape: AttnShape, q_gamma: torch.Tensor,
                      k_gamma: torch.Tensor, cs: torch.Tensor, ws: DecodeWorkspace, scale: float | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Fused paged step: per sequence s, norm+RoPE at position kv_len[s]-1, append to its
    physical row, attention over its kv_len[s] keys.  qkv [n_seq, (H+2HKV)*128]."""
    _need_gpu_f32("qkv", qkv)
    n_seq, max_blocks = block_table.shape
    out = torch.empty((n_seq, shape.n_head, HEAD_DIM), dtype=torch.float32, device=qkv.device) if out is None else out
    scale = default_scale() if scale is None else scale
    _capi.call("ei_decode_step_paged", _stream(), qkv.data_ptr(), qkv.stride(0), out.data_ptr(), kc.data_ptr(),
               vc.data_ptr(), block_table.data_ptr(), max_blocks, block_size, kv_len.data_ptr(), n_seq, shape.n_head,
               shape.n_head_kv, shape.head_dim, q_gamma.data_ptr(), k_gamma.data_ptr(), cs.data_ptr(),
               shape.rope_dim, float(shape.eps), float(scale), ws.max_kv, ws.buf.data_ptr(), ws.nbytes)
    return out


# ---------------------------------------------------------------- prefill
class PrefillWorkspace:
    """Key-split shares for ei_attn_prefill_split / ei_prefill_step: serves chunks of up to max_B
    rows with pos0 + B <= max_kv (max_kv only steers the split plan; larger positions stay correct)."""

    def __init__(self, max_B: int, n_head: int, n_head_kv: int, max_kv: int, device="cuda"):
        self.max_B, self.max_kv = max_B, max_kv
        self.nbytes = int(_capi.lib().ei_attn_prefill_ws_bytes(max_B, n_head, n_head_kv, max_kv))
        self.buf = torch.empty(max(self.nbytes, 256), dtype=torch.uint8, device=device)


def attn_prefill(q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, pos_dev: torch.Tensor, shape: AttnShape,
                 B: int | None = None, scale: float | None = None, out: torch.Tensor | None = None,
                 ws: PrefillWorkspace | None = None) -> torch.Tensor:
    """q rows [B, >= H*128] (normed + roped, heads first); returns [B, H, 128].
    With `ws` the key range is split over workgroups for short chunks (ei_attn_prefill_split)."""
    _need_gpu_f32("q", q)
    B = q.shape[0] if B is None else B
    out = torch.empty((B, shape.n_head, HEAD_DIM), dtype=torch.float32, device=q.device) if out is None else out
    scale = default_scale() if scale is None else scale
    if ws is None:
        _capi.call("ei_attn_prefill", _stream(), q.data_ptr(), q.stride(0), out.data_ptr(), kc.data_ptr(),
                   vc.data_ptr(), pos_dev.data_ptr(), B, shape.n_head, shape.n_head_kv, shape.head_dim, float(scale))
    else:
        if B > ws.max_B:
            raise ValueError(f"prefill workspace serves chunks of up to {ws.max_B} rows, got B={B}")
        _capi.call("ei_attn_prefill_split", _stream(), q.data_ptr(), q.stride(0), out.data_ptr(), kc.data_ptr(),
                   vc.data_ptr(), pos_dev.data_ptr(), B, shape.n_head, shape.n_head_kv, shape.head_dim, float(scale),
                   ws.max_kv, ws.buf.data_ptr(), ws.nbytes)
    return out


def prefill_step(qkv: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, shape: AttnShape, q_gamma: torch.Tensor,
                 k_gamma: torch.Tensor, cs: torch.Tensor, pos_dev: torch.Tensor, ws: PrefillWorkspace,
                 B: int | None = None, scale: float | None = None, out: torch.Tensor | None = None,
                 block_table: torch.Tensor | None = None, block_size: int = 0) -> torch.Tensor:
    """Fused chunk step (ei_prefill_step): K heads normed + roped in place and appended with V
    at rows pos..pos+B-1; Q heads left raw in qkv and normed inside the attention kernel.
    qkv [B, >= (H+2HKV)*128]; returns [B, H, 128].  With block_table (int32 [max_blocks]) the
    caches are a paged pool of block_size-row blocks (ei_prefill_step_paged)."""
    _need_gpu_f32("qkv", qkv)
    B = qkv.shape[0] if B is None else B
    if B > ws.max_B:
        raise ValueError(f"prefill workspace serves chunks of up to {ws.max_B} rows, got B={B}")
    out = torch.empty((B, shape.n_head, HEAD_DIM), dtype=torch.float32, device=qkv.device) if out is None else out
    scale = default_scale() if scale is None else scale
    tail = (q_gamma.data_ptr(), k_gamma.data_ptr(), cs.data_ptr(), shape.rope_dim, float(shape.eps), float(scale),
            ws.max_kv, ws.buf.data_ptr(), ws.nbytes)
    if block_table is None:
        _capi.call("ei_prefill_step", _stream(), qkv.data_ptr(), qkv.stride(0), out.data_ptr(), kc.data_ptr(),
                   vc.data_ptr(), pos_dev.data_ptr(), B, shape.n_head, shape.n_head_kv, shape.head_dim, *tail)
    else:
        _capi.call("ei_prefill_step_paged", _stream(), qkv.data_ptr(), qkv.stride(0), out.data_ptr(), kc.data_ptr(),
                   vc.data_ptr(), block_table.data_ptr(), block_table.numel(), block_size, pos_dev.data_ptr(), B,
                   shape.n_head, shape.n_head_kv, shape.head_dim, *tail)
    return out


# ---------------------------------------------------------------- rotary positions of packed rows
_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}
_LAYOUTS = {"half": 0, "interleaved": 1}


@dataclass(frozen=True)
class RopeScaling:
    """How the rotary frequencies are scaled for contexts `factor` times as long as the n_trained
    positions a model was trained for (include/ei_packed.h): none, linear, ntk or yarn."""

    kind: str = "none"
    factor: float = 1.0
    n_trained: int = 0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attn_factor: float = 0.0  # yarn: factor on cos and sin, 0: 0.1 ln(factor) + 1


def _device() -> int:
    """The current device, on whose current stream a call is launched."""
    return torch._C._cuda_getDevice()  # (torch.cuda.current_device() checks for a context first: 0.1 us)


def _refuse(name: str, t: torch.Tensor, dtype: torch.dtype) -> None:
    """Says why a tensor that failed a check is not one of this dtype on the current device."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"{name} is on {t.device}, the current device is cuda:{torch.cuda.current_device()}")


def _need_contiguous(name: str, t: torch.Tensor, dtype: torch.dtype) -> None:
    if t.dtype is not dtype or t.get_device() != _device() or not t.is_contiguous():
        _refuse(name, t, dtype)
        raise ValueError(f"{name} must be contiguous")


def _need_gamma(name: str, t: torch.Tensor | None) -> None:
    if t is not None:
        _need_contiguous(name, t, torch.float32)
        if t.numel() != HEAD_DIM:
            raise ValueError(f"{name} must hold {HEAD_DIM} values, got {t.numel()}")


def _rows_of(name: str, t: torch.Tensor, rows: int, width: int) -> int:
    """Row stride of a [>= rows, >= width] matrix (or [>= rows, heads, 128]), after checking it."""
    shape, stride = t.shape, t.stride()
    if t.dtype is not torch.float32 or t.get_device() != _device():
        _refuse(name, t, torch.float32)
    if len(shape) == 2:
        have = shape[1]
    elif len(shape) == 3 and (stride[1] == shape[2] or shape[1] == 1):
        have = shape[1] * shape[2]
    else:
        raise ValueError(f"{name} must be [rows, values] or [rows, heads, {HEAD_DIM}] with whole rows")
    if stride[-1] != 1 and t.numel():
        raise ValueError(f"{name} must be contiguous in its last dimension")
    if shape[0] < rows or have < width:
        raise ValueError(f"{name} must hold {rows} rows of {width} values, got {tuple(shape)}")
    return stride[0] if shape[0] > 1 else width  # (a single row's stride is whatever the view says)


def rope_table_scaled(n_pos: int, rope_dim: int = HEAD_DIM, theta: float = 1e6, scaling: RopeScaling | None = None,
                      out: torch.Tensor | None = None, device="cuda") -> torch.Tensor:
    """[n_pos, rope_dim/2, 2] (cos, sin) table made on the GPU, angles in double, for plain or scaled
    frequencies (ei_rope_table_scaled).  It serves every function that takes a table."""
    import ctypes
    sc = scaling or RopeScaling()
    if sc.kind not in _SCALINGS:
        raise ValueError(f"scaling kind {sc.kind!r}: one of {', '.join(_SCALINGS)}")
    if out is None:
        out = torch.empty((n_pos, rope_dim // 2, 2), dtype=torch.float32, device=device)
    _need_contiguous("out", out, torch.float32)
    if out.shape != (n_pos, rope_dim // 2, 2):
        raise ValueError(f"out must be [{n_pos}, {rope_dim // 2}, 2], got {tuple(out.shape)}")
    c = _capi.RopeScalingC(_SCALINGS[sc.kind], sc.factor, sc.n_trained, sc.beta_fast, sc.beta_slow, sc.attn_factor)
    _capi.call("ei_rope_table_scaled", _stream(), out.data_ptr(), n_pos, rope_dim, float(theta), ctypes.byref(c))
    return out


def _table_positions(cs: torch.Tensor, rope_dim: int) -> int:
    _need_contiguous("cs", cs, torch.float32)
    shape = cs.shape
    if len(shape) != 3 or shape[1] != rope_dim // 2 or shape[2] != 2:
        raise ValueError(f"cs must be [positions, {rope_dim // 2}, 2], got {tuple(shape)}")
    return shape[0]


def rope_rows(x: torch.Tensor, n_heads: int, cs: torch.Tensor, pos: torch.Tensor, rope_dim: int = HEAD_DIM,
              layout: str = "half", gamma: torch.Tensor | None = None, eps: float = 1e-6,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """Turns the first n_heads heads of each row of x [rows, >= n_heads*128] to the row's position
    pos (int32 [rows]), normed first when gamma is given (ei_rope_rows).  Into `out`, which may be x;
    a row whose position lies outside the table is copied as it is."""
    if layout not in _LAYOUTS:
        raise ValueError(f"layout {layout!r}: one of {', '.join(_LAYOUTS)}")
    _need_contiguous("pos", pos, torch.int32)
    _need_gamma("gamma", gamma)
    rows, width = pos.numel(), n_heads * HEAD_DIM
    xs = _rows_of("x", x, rows, width)
    if out is None:
        out = torch.empty((rows, width), dtype=torch.float32, device=x.device)
    ys, n_pos = _rows_of("out", out, rows, width), _table_positions(cs, rope_dim)
    if rows:  # (an empty tensor has no address)
        _capi.call("ei_rope_rows", _stream(), x.data_ptr(), xs, out.data_ptr(), ys, rows, n_heads, HEAD_DIM,
                   _ptr(gamma), float(eps), cs.data_ptr(), n_pos, pos.data_ptr(), rope_dim, _LAYOUTS[layout])
    return out


# ---------------------------------------------------------------- several sequences' rows in one call
class PackedBatch:
    """Plan and workspace of batches of up to max_seq sequences and max_rows new rows
    (include/ei_packed.h).  plan() lays a batch out from its lengths, once for all layers; the calls
    that take the batch then run one after another (they share the workspace)."""

    def __init__(self, max_seq: int, max_rows: int, n_head: int, n_head_kv: int, device="cuda"):
        self.max_seq, self.max_rows, self.n_head, self.n_head_kv = max_seq, max_rows, n_head, n_head_kv
        self.nbytes = int(_capi.lib().ei_packed_plan_bytes(max_seq, max_rows, n_head, n_head_kv))
        self.ws_nbytes = int(_capi.lib().ei_packed_ws_bytes(max_rows, n_head, n_head_kv))
        if self.nbytes == 0 or self.ws_nbytes == 0:
            raise ValueError("invalid packed batch shape")
        self.buf = torch.empty(self.nbytes, dtype=torch.uint8, device=device)
        self.ws = torch.empty(self.ws_nbytes, dtype=torch.uint8, device=device)
        self._device = self.buf.get_device()
        self.n_seq = 0  # no plan yet
        self.rows = 0
        self.prompts = False

    def plan(self, cu_rows: torch.Tensor, rows: int, max_kv: int, kv_len: torch.Tensor | None = None) -> None:
        """cu_rows int32 [n_seq + 1]: sequence s owns rows cu_rows[s] .. cu_rows[s+1] - 1, of `rows` in
        all (later ones belong to nobody).  kv_len int32 [n_seq], each at most max_kv: keys after the
        new rows are appended; None: whole prompts, of at most max_kv rows each."""
        self._check_device()
        _need_contiguous("cu_rows", cu_rows, torch.int32)
        n_seq = cu_rows.numel() - 1
        if not 1 <= n_seq <= self.max_seq or not 0 <= rows <= self.max_rows:
            raise ValueError(f"batch of {n_seq} sequences and {rows} rows: made for 1 to {self.max_seq} sequences and "
                             f"up to {self.max_rows} rows")
        if not 0 <= max_kv <= 1 << 30:  # (ctypes would cut it to 32 bits)
            raise ValueError(f"max_kv {max_kv} out of range [0, 2^30]")
        if kv_len is not None:
            _need_contiguous("kv_len", kv_len, torch.int32)
            if kv_len.numel() != n_seq:
                raise ValueError(f"kv_len must hold {n_seq} lengths, got {kv_len.numel()}")
        _capi.call("ei_packed_plan", _stream(), cu_rows.data_ptr(), _ptr(kv_len), n_seq, rows, max_kv, self.n_head,
                   self.n_head_kv, self.buf.data_ptr(), self.nbytes)
        self.n_seq, self.rows, self.prompts = n_seq, rows, kv_len is None

    def _check_device(self) -> None:
        if self.buf.get_device() != _device():
            _refuse("the batch's plan", self.buf, torch.uint8)

    def _check(self, shape: AttnShape) -> None:
        if self.n_seq == 0:
            raise ValueError("the batch has no plan yet: call plan() first")
        self._check_device()
        if (shape.n_head, shape.n_head_kv) != (self.n_head, self.n_head_kv):
            raise ValueError(f"the batch was made for {self.n_head}/{self.n_head_kv} heads, the call has "
                             f"{shape.n_head}/{shape.n_head_kv}")

    def _out(self, out: torch.Tensor | None, device) -> torch.Tensor:
        if out is None:
            return torch.empty((self.rows, self.n_head, HEAD_DIM), dtype=torch.float32, device=device)
        _need_contiguous("out", out, torch.float32)
        if out.numel() < self.rows * self.n_head * HEAD_DIM:
            raise ValueError(f"out must hold {self.rows} rows of {self.n_head * HEAD_DIM} values")
        return out

    def _tail(self) -> tuple:
        return self.buf.data_ptr(), self.nbytes, self.ws.data_ptr(), self.ws_nbytes


def attn_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, batch: PackedBatch, shape: AttnShape,
                scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of whole prompts packed one after another (ei_attn_packed): q [rows, >= H*128],
    k and v [rows, >= HKV*128] (normed and turned; views of one buffer are fine), batch planned without
    kv_len; returns [rows, H, 128]."""
    batch._check(shape)
    if not batch.prompts:
        raise ValueError("the batch is planned over a cache (kv_len): attn_packed takes whole prompts")
    qs = _rows_of("q", q, batch.rows, shape.n_head * HEAD_DIM)
    ks, vs = _rows_of("k", k, batch.rows, shape.kd), _rows_of("v", v, batch.rows, shape.kd)
    if ks != vs:
        raise ValueError(f"k and v must share a row stride, got {ks} and {vs}")
    out = batch._out(out, q.device)
    scale = default_scale() if scale is None else scale
    if batch.rows == 0:
        return out
    _capi.call("ei_attn_packed", _stream(), q.data_ptr(), qs, k.data_ptr(), v.data_ptr(), ks, out.data_ptr(),
               batch.n_seq, batch.rows, shape.n_head, shape.n_head_kv, shape.head_dim, float(scale), *batch._tail())
    return out


def _pool_args(kc: torch.Tensor, vc: torch.Tensor, block_table: torch.Tensor, block_size: int, batch: PackedBatch,
               shape: AttnShape) -> tuple:
    for name, t in (("kc", kc), ("vc", vc)):
        _need_contiguous(name, t, torch.float32)
    if kc.numel() != vc.numel() or kc.numel() % shape.kd:
        raise ValueError(f"kc and vc must be pools of rows of {shape.kd} values, got {tuple(kc.shape)} and "
                         f"{tuple(vc.shape)}")
    _need_contiguous("block_table", block_table, torch.int32)
    if block_table.dim() != 2 or block_table.shape[0] < batch.n_seq:
        raise ValueError(f"block_table must be [{batch.n_seq}, blocks], got {tuple(block_table.shape)}")
    if block_size <= 0:
        raise ValueError(f"block_size {block_size} must be positive")
    return (kc.data_ptr(), vc.data_ptr(), kc.numel() // shape.kd // block_size, block_table.data_ptr(),
            block_table.shape[1], block_size)


def attn_packed_paged(q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, block_table: torch.Tensor, block_size: int,
                      batch: PackedBatch, shape: AttnShape, scale: float | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the batch's new rows, q [rows, >= H*128] normed and turned, over each sequence's pages
    of the pool kc, vc (their new keys already there; block_table int32 [n_seq, blocks]): a chunk of a
    prompt, draft tokens or a single token each (ei_attn_packed_paged).  Returns [rows, H, 128]."""
    batch._check(shape)
    qs = _rows_of("q", q, batch.rows, shape.n_head * HEAD_DIM)
    pool = _pool_args(kc, vc, block_table, block_size, batch, shape)
    out = batch._out(out, q.device)
    scale = default_scale() if scale is None else scale
    if batch.rows == 0:
        return out
    _capi.call("ei_attn_packed_paged", _stream(), q.data_ptr(), qs, out.data_ptr(), *pool, batch.n_seq, batch.rows,
               shape.n_head, shape.n_head_kv, shape.head_dim, float(scale), *batch._tail())
    return out


def packed_step_paged(qkv: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, block_table: torch.Tensor,
                      block_size: int, batch: PackedBatch, shape: AttnShape, q_gamma: torch.Tensor,
                      k_gamma: torch.Tensor, cs: torch.Tensor, scale: float | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """The whole step of a batch from raw projections qkv [rows, >= (H+2HKV)*128], which it only reads:
    QK-norm and rotary positions, K and V appended to the sequences' pages, attention
    (ei_packed_step_paged).  Returns [rows, H, 128]."""
    batch._check(shape)
    rs = _rows_of("qkv", qkv, batch.rows, shape.qkv)
    pool = _pool_args(kc, vc, block_table, block_size, batch, shape)
    _need_gamma("q_gamma", q_gamma)
    _need_gamma("k_gamma", k_gamma)
    n_pos = _table_positions(cs, shape.rope_dim)
    out = batch._out(out, qkv.device)
    scale = default_scale() if scale is None else scale
    if batch.rows == 0:
        return out
    _capi.call("ei_packed_step_paged", _stream(), qkv.data_ptr(), rs, out.data_ptr(), *pool, batch.n_seq, batch.rows,
               shape.n_head, shape.n_head_kv, shape.head_dim, q_gamma.data_ptr(), k_gamma.data_ptr(), cs.data_ptr(),
               n_pos, shape.rope_dim, float(shape.eps), float(scale), *batch._tail())
    return out


# ---------------------------------------------------------------- 8-bit cache, trees of drafted tokens
_CACHE_KINDS = {"e4m3": (1, torch.float8_e4m3fn), "int8": (2, torch.int8)}


class Cache8:
    """A paged pool of 8-bit keys and values (include/ei_cache8.h): codes k, v [n_blocks, HKV, block_size, 128]
    (float8_e4m3fn or int8) and scales k_scale, v_scale [n_blocks, HKV, block_size]; a code stands for
    code * scale.  Made empty (zeros), or of tensors that a program has already; calls read the tensors' addresses each
    time, the tensors themselves stay those it was made of."""

    def __init__(self, n_blocks: int, block_size: int, n_head_kv: int, kind: str = "e4m3", device="cuda"):
        if kind not in _CACHE_KINDS:
            raise ValueError(f"cache kind {kind!r}: one of {', '.join(_CACHE_KINDS)}")
        shape = (n_blocks, n_head_kv, block_size)
        codes = [torch.zeros((*shape, HEAD_DIM), dtype=torch.int8, device=device).view(_CACHE_KINDS[kind][1])
                 for _ in range(2)]
        self._take(*codes, *(torch.zeros(shape, dtype=torch.float32, device=device) for _ in range(2)))

    @classmethod
    def of(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> "Cache8":
        cache = cls.__new__(cls)
        cache._take(k, v, k_scale, v_scale)
        return cache

    def _take(self, k, v, k_scale, v_scale) -> None:
        kinds = {dtype: (name, number) for name, (number, dtype) in _CACHE_KINDS.items()}
        if k.dtype not in kinds:
            raise ValueError(f"codes must be torch.float8_e4m3fn or torch.int8, got {k.dtype}")
        if k.dim() != 4 or k.shape[-1] != HEAD_DIM:
            raise ValueError(f"codes must be [blocks, KV heads, block size, {HEAD_DIM}], got {tuple(k.shape)}")
        for name, t, shape, dtype in (("k", k, k.shape, k.dtype), ("v", v, k.shape, k.dtype),
                                      ("k_scale", k_scale, k.shape[:3], torch.float32),
                                      ("v_scale", v_scale, k.shape[:3], torch.float32)):
            if t.dtype is not dtype or t.shape != shape or not t.is_contiguous() or t.device != k.device:
                raise ValueError(f"{name} must be a contiguous {dtype} tensor {tuple(shape)} on {k.device}, got "
                                 f"{t.dtype} {tuple(t.shape)} on {t.device}")
        import ctypes
        self._tensors = k, v, k_scale, v_scale
        self._kind, number = kinds[k.dtype]
        self._shape = n_blocks, _, block_size = k.shape[:3]
        self._at = k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr()
        self._c = _capi.Cache8C(*self._at, number, n_blocks, block_size)
        self._c_at = ctypes.addressof(self._c)
        self._device = k.get_device()

    k, v, k_scale, v_scale = (property(lambda self, i=i: self._tensors[i]) for i in range(4))
    n_blocks, n_head_kv, block_size = (property(lambda self, i=i: self._shape[i]) for i in range(3))
    kind = property(lambda self: self._kind)

    def _address(self) -> int:
        """Of the ei_cache8 that the tensors are now."""
        k, v, k_scale, v_scale = self._tensors
        if (k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr()) != self._at:
            self._take(k, v, k_scale, v_scale)
        return self._c_at


# (A call's launch takes 4 us of host time; its checks, with a function and a message for each, took as much again.  So
# each tensor's properties are asked for once, on the device `dev` that was asked for once, and what is wrong is found
# out where something is.)
def _check_batch(batch: PackedBatch, shape: AttnShape, dev: int) -> None:
    if (batch.n_seq == 0 or batch._device != dev or batch.n_head != shape.n_head or
            batch.n_head_kv != shape.n_head_kv):
        batch._check(shape)


def _check_planned(batch: PackedBatch, dev: int) -> None:
    if batch.n_seq == 0:
        raise ValueError("the batch has no plan yet: call plan() first")
    if batch._device != dev:
        batch._check_device()


def _stride_of(name: str, t: torch.Tensor, rows: int, width: int, dev: int) -> int:
    """_rows_of, for the usual matrix."""
    shape, stride = t.shape, t.stride()
    if (len(shape) == 2 and shape[0] >= rows and shape[0] > 1 and shape[1] >= width and stride[1] == 1 and
            t.dtype is torch.float32 and t.get_device() == dev):
        return stride[0]
    return _rows_of(name, t, rows, width)


def _out_of(batch: PackedBatch, out: torch.Tensor | None, dev: int) -> torch.Tensor:
    if (out is not None and out.dtype is torch.float32 and out.get_device() == dev and
            out.numel() >= batch.rows * batch.n_head * HEAD_DIM and out.is_contiguous()):
        return out
    return batch._out(out, batch.buf.device)


def _cache8_args(cache: Cache8, block_table: torch.Tensor, batch: PackedBatch, n_head_kv: int, dev: int) -> tuple:
    at = cache._address()
    if cache._shape[1] != n_head_kv:
        raise ValueError(f"the cache holds {cache.n_head_kv} KV heads, the call has {n_head_kv}")
    if cache._device != dev:
        _refuse("the cache", cache.k, cache.k.dtype)
    shape = block_table.shape
    if (block_table.dtype is not torch.int32 or block_table.get_device() != dev or len(shape) != 2 or
            shape[0] < batch.n_seq or not block_table.is_contiguous()):
        _need_contiguous("block_table", block_table, torch.int32)
        raise ValueError(f"block_table must be [{batch.n_seq}, blocks], got {tuple(shape)}")
    return at, block_table.data_ptr(), shape[1]


def _pool_of(kc: torch.Tensor, vc: torch.Tensor, block_table: torch.Tensor, block_size: int, batch: PackedBatch,
             shape: AttnShape, dev: int) -> tuple:
    """_pool_args, for what passes its checks."""
    f32, n, table, kd = torch.float32, kc.numel(), block_table.shape, shape.kd
    if (kc.dtype is f32 and vc.dtype is f32 and kc.get_device() == dev and vc.get_device() == dev and
            kc.is_contiguous() and vc.is_contiguous() and n == vc.numel() and n % kd == 0 and len(table) == 2 and
            table[0] >= batch.n_seq and block_table.dtype is torch.int32 and block_table.get_device() == dev and
            block_table.is_contiguous() and block_size > 0):
        return kc.data_ptr(), vc.data_ptr(), n // kd // block_size, block_table.data_ptr(), table[1], block_size
    return _pool_args(kc, vc, block_table, block_size, batch, shape)


def _mask_args(mask: torch.Tensor | None, rows: int) -> tuple:
    if mask is None:
        return None, 0
    shape = mask.shape
    if mask.dtype is not torch.int64 or mask.get_device() != _device() or not mask.is_contiguous():
        _need_contiguous("mask", mask, torch.int64)
    if len(shape) != 2 or shape[0] < rows or shape[1] < 1:
        raise ValueError(f"mask must be [{rows}, words], got {tuple(shape)}")
    return mask.data_ptr(), shape[1]


def _turn_args(cs: torch.Tensor, pos: torch.Tensor | None, shape: AttnShape, rows: int, q_gamma: torch.Tensor,
               k_gamma: torch.Tensor, dev: int) -> tuple:
    """q_gamma, k_gamma, cs, n_pos, turn_at, rope_dim, eps."""
    f32 = torch.float32
    for name, t in (("q_gamma", q_gamma), ("k_gamma", k_gamma)):
        if t is None:
            raise ValueError(f"{name} is missing")
        if t.dtype is not f32 or t.get_device() != dev or t.numel() != HEAD_DIM or not t.is_contiguous():
            _need_gamma(name, t)
    table = cs.shape
    if (len(table) != 3 or table[1] != shape.rope_dim // 2 or table[2] != 2 or cs.dtype is not f32 or
            cs.get_device() != dev or not cs.is_contiguous()):
        _table_positions(cs, shape.rope_dim)
    if pos is not None:
        _need_contiguous("pos", pos, torch.int32)
        if pos.numel() < rows:
            raise ValueError(f"pos must hold {rows} positions, got {pos.numel()}")
        pos = pos.data_ptr()
    return q_gamma.data_ptr(), k_gamma.data_ptr(), cs.data_ptr(), table[0], pos, shape.rope_dim, shape.eps


def cache8_store(qkv: torch.Tensor, cache: Cache8, block_table: torch.Tensor, batch: PackedBatch, shape: AttnShape,
                 q_gamma: torch.Tensor, k_gamma: torch.Tensor, cs: torch.Tensor, pos: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Norms, turns and quantises the batch's new rows from raw projections qkv [rows, >= (H+2HKV)*128] into their
    sequences' pages, and returns the normed and turned queries [rows, H, 128] (ei_cache8_store).  pos
    int32 [rows]: positions other than the rows' slots, as of a tree's tokens."""
    dev = _device()
    _check_batch(batch, shape, dev)
    rs = _stride_of("qkv", qkv, batch.rows, shape.qkv, dev)
    where = _cache8_args(cache, block_table, batch, shape.n_head_kv, dev)
    turn = _turn_args(cs, pos, shape, batch.rows, q_gamma, k_gamma, dev)
    out = _out_of(batch, out, dev)
    if batch.rows:
        _capi.call("ei_cache8_store", _stream_on(dev), qkv.data_ptr(), rs, out.data_ptr(), *where, batch.n_seq,
                   batch.rows, shape.n_head, shape.n_head_kv, shape.head_dim, *turn, batch.buf.data_ptr(),
                   batch.nbytes)
    return out


def cache8_load(cache: Cache8, block_table: torch.Tensor, batch: PackedBatch,
                out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The cached keys and values of the batch's new rows in 32 bits, [rows, HKV, 128] each (ei_cache8_load); a batch
    planned with longer runs of rows reads more of the sequences.  out: two tensors of one row stride."""
    dev = _device()
    _check_planned(batch, dev)
    where = _cache8_args(cache, block_table, batch, batch.n_head_kv, dev)
    width = cache.n_head_kv * HEAD_DIM
    if out is None:
        out = tuple(torch.empty((batch.rows, cache.n_head_kv, HEAD_DIM), dtype=torch.float32, device=cache.k.device)
                    for _ in range(2))
    k, v = out
    ks, vs = _rows_of("out[0]", k, batch.rows, width), _rows_of("out[1]", v, batch.rows, width)
    if ks != vs:
        raise ValueError(f"the two outputs must share a row stride, got {ks} and {vs}")
    if batch.rows:
        _capi.call("ei_cache8_load", _stream_on(dev), *where, k.data_ptr(), v.data_ptr(), ks, batch.n_seq, batch.rows,
                   batch.n_head, batch.n_head_kv, HEAD_DIM, batch.buf.data_ptr(), batch.nbytes)
    return k, v


def attn_packed_cache8(q: torch.Tensor, cache: Cache8, block_table: torch.Tensor, batch: PackedBatch, shape: AttnShape,
                       mask: torch.Tensor | None = None, scale: float | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the batch's new rows, q [rows, >= H*128] normed and turned, over their sequences' pages of the
    8-bit cache (ei_attn_packed_cache8): causal, or with mask (int64 [rows, words]) a row sees of the new rows
    those whose bit is set in its words, up to itself.  Returns [rows, H, 128]."""
    dev = _device()
    _check_batch(batch, shape, dev)
    qs = _stride_of("q", q, batch.rows, shape.n_head * HEAD_DIM, dev)
    where = _cache8_args(cache, block_table, batch, shape.n_head_kv, dev)
    bits = _mask_args(mask, batch.rows)
    out = _out_of(batch, out, dev)
    scale = _SCALE if scale is None else float(scale)
    if batch.rows:
        _capi.call("ei_attn_packed_cache8", _stream_on(dev), q.data_ptr(), qs, out.data_ptr(), *where, batch.n_seq,
                   batch.rows, shape.n_head, shape.n_head_kv, shape.head_dim, *bits, scale, *batch._tail())
    return out


def packed_step_cache8(qkv: torch.Tensor, cache: Cache8, block_table: torch.Tensor, batch: PackedBatch,
                       shape: AttnShape, q_gamma: torch.Tensor, k_gamma: torch.Tensor, cs: torch.Tensor,
                       pos: torch.Tensor | None = None, mask: torch.Tensor | None = None, scale: float | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """The whole step of a batch over the 8-bit cache: cache8_store, then attn_packed_cache8 on its queries
    (ei_packed_step_cache8).  Returns [rows, H, 128]."""
    dev = _device()
    _check_batch(batch, shape, dev)
    rs = _stride_of("qkv", qkv, batch.rows, shape.qkv, dev)
    where = _cache8_args(cache, block_table, batch, shape.n_head_kv, dev)
    turn = _turn_args(cs, pos, shape, batch.rows, q_gamma, k_gamma, dev)
    bits = _mask_args(mask, batch.rows)
    out = _out_of(batch, out, dev)
    scale = _SCALE if scale is None else float(scale)
    if batch.rows:
        _capi.call("ei_packed_step_cache8", _stream_on(dev), qkv.data_ptr(), rs, out.data_ptr(), *where, batch.n_seq,
                   batch.rows, shape.n_head, shape.n_head_kv, shape.head_dim, *turn, *bits, scale, *batch._tail())
    return out


def attn_tree_paged(q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, block_table: torch.Tensor, block_size: int,
                    batch: PackedBatch, shape: AttnShape, mask: torch.Tensor, scale: float | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """attn_packed_paged for trees of drafted tokens (ei_attn_tree_paged): a row sees the keys before its sequence's
    new rows, and of those the ones whose bit is set in its row of mask (int64 [rows, words]), up to itself."""
    dev = _device()
    _check_batch(batch, shape, dev)
    qs = _stride_of("q", q, batch.rows, shape.n_head * HEAD_DIM, dev)
    pool = _pool_of(kc, vc, block_table, block_size, batch, shape, dev)
    bits = _mask_args(mask, batch.rows)
    out = _out_of(batch, out, dev)
    scale = _SCALE if scale is None else float(scale)
    if batch.rows:
        _capi.call("ei_attn_tree_paged", _stream_on(dev), q.data_ptr(), qs, out.data_ptr(), *pool, batch.n_seq,
                   batch.rows, shape.n_head, shape.n_head_kv, shape.head_dim, *bits, scale, *batch._tail())
    return out


def tree_step_paged(qkv: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, block_table: torch.Tensor, block_size: int,
                    batch: PackedBatch, shape: AttnShape, q_gamma: torch.Tensor, k_gamma: torch.Tensor,
                    cs: torch.Tensor, pos: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                    scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """packed_step_paged for trees of drafted tokens, at positions pos (int32 [rows], None: the rows' slots) and with
    a mask (ei_tree_step_paged).  Returns [rows, H, 128]."""
    dev = _device()
    _check_batch(batch, shape, dev)
    rs = _stride_of("qkv", qkv, batch.rows, shape.qkv, dev)
    pool = _pool_of(kc, vc, block_table, block_size, batch, shape, dev)
    turn = _turn_args(cs, pos, shape, batch.rows, q_gamma, k_gamma, dev)
    bits = _mask_args(mask, batch.rows)
    out = _out_of(batch, out, dev)
    scale = _SCALE if scale is None else float(scale)
    if batch.rows:
        _capi.call("ei_tree_step_paged", _stream_on(dev), qkv.data_ptr(), rs, out.data_ptr(), *pool, batch.n_seq,
                   batch.rows, shape.n_head, shape.n_head_kv, shape.head_dim, *turn, *bits, scale, *batch._tail())
    return out


def _kept_args(batch: PackedBatch, kept: torch.Tensor, n_kept: torch.Tensor, out: torch.Tensor | None,
               dev: int) -> tuple:
    shape, n_seq, i32 = kept.shape, batch.n_seq, torch.int32
    if (len(shape) != 2 or shape[0] < n_seq or shape[1] < 1 or kept.dtype is not i32 or kept.get_device() != dev or
            not kept.is_contiguous()):
        _need_contiguous("kept", kept, i32)
        raise ValueError(f"kept must be [{n_seq}, most], got {tuple(shape)}")
    if out is None:
        out = torch.empty(n_seq, dtype=i32, device=kept.device)
    for name, t in (("n_kept", n_kept), ("out", out)):
        if t.dtype is not i32 or t.get_device() != dev or t.numel() < n_seq or not t.is_contiguous():
            _need_contiguous(name, t, i32)
            raise ValueError(f"{name} must hold {n_seq} numbers, got {t.numel()}")
    return (kept.data_ptr(), shape[1], n_kept.data_ptr(), out.data_ptr(), batch.buf.data_ptr(), batch.nbytes), out


def cache_keep(kc: torch.Tensor, vc: torch.Tensor, block_table: torch.Tensor, block_size: int, batch: PackedBatch,
               shape: AttnShape, kept: torch.Tensor, n_kept: torch.Tensor,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """After a batch of drafts was checked: moves the accepted rows of each sequence's new rows, kept int32
    [n_seq, most] (rising; n_kept int32 [n_seq] of them count), together behind its earlier keys in the fp32 pool
    (ei_cache_keep).  Returns the sequences' lengths with them, int32 [n_seq]; `out` may be the batch's kv_len."""
    dev = _device()
    _check_batch(batch, shape, dev)
    pool = _pool_of(kc, vc, block_table, block_size, batch, shape, dev)
    args, out = _kept_args(batch, kept, n_kept, out, dev)
    _capi.call("ei_cache_keep", _stream_on(dev), *pool, batch.n_seq, batch.rows, shape.n_head, shape.n_head_kv,
               shape.head_dim, *args)
    return out


def cache8_keep(cache: Cache8, block_table: torch.Tensor, batch: PackedBatch, kept: torch.Tensor, n_kept: torch.Tensor,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """cache_keep in the 8-bit cache (ei_cache8_keep)."""
    dev = _device()
    _check_planned(batch, dev)
    where = _cache8_args(cache, block_table, batch, batch.n_head_kv, dev)
    args, out = _kept_args(batch, kept, n_kept, out, dev)
    _capi.call("ei_cache8_keep", _stream_on(dev), *where, batch.n_seq, batch.rows, batch.n_head, batch.n_head_kv,
               HEAD_DIM, *args)
    return out


# ---------------------------------------------------------------- synthetic inputs
def synth_fill(t: torch.Tensor, seed: int, offset: int = 0, row_len: int = 1, spike_every: int = 0,
               spike_mult: float = 1.0) -> torch.Tensor:
    """Fill a contiguous float32 GPU tensor with the counter-based N(0,1) stream (in place)."""
    _need_gpu_f32("t", t)
    if not t.is_contiguous():
        raise ValueError("t must be contiguous")
    _capi.call("ei_synth_fill", _stream(), t.data_ptr(), t.numel(), seed, offset, row_len, spike_every,
               float(spike_mult))
    return t


def flops_causal(T_new: int, pos0: int, n_head: int, head_dim: int = HEAD_DIM) -> float:
    """Algorithmic FLOPs of causal attention: 4*D per visible (query, key) pair, per head."""
    pairs = sum(pos0 + b + 1 for b in range(T_new)) if T_new < 64 else T_new * pos0 + T_new * (T_new + 1) // 2
    return 4.0 * head_dim * pairs * n_head


def decode_bytes(kv_len: int, n_head: int, n_head_kv: int, head_dim: int = HEAD_DIM) -> float:
    """Algorithmic HBM bytes of one decode: the visible K and V rows plus q and out."""
    return 4.0 * (2 * kv_len * n_head_kv * head_dim + 2 * n_head * head_dim)


__all__ = [
    "AttnShape", "DecodeWorkspace", "attn_decode", "attn_decode_batched", "attn_prefill", "decode_step",
    "default_scale", "headnorm_rope", "kv_append", "qkv_prepare", "rope_table", "synth_fill", "flops_causal",
    "decode_bytes", "RopeScaling", "rope_table_scaled", "rope_rows", "PackedBatch", "attn_packed",
    "attn_packed_paged", "packed_step_paged", "Cache8", "cache8_store", "cache8_load", "attn_packed_cache8",
    "packed_step_cache8", "attn_tree_paged", "tree_step_paged", "cache_keep", "cache8_keep",
]
