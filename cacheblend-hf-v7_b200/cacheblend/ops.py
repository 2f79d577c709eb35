"""torch-facing wrappers of the libcbk kernels.

Each wrapper validates devices, dtypes, shapes and contiguity, passes raw
device pointers plus the current CUDA stream to the C ABI, and maps return
codes to Python exceptions.  Nothing here runs on the CPU: a non-CUDA tensor is
an error.
"""
from __future__ import annotations

import ctypes
import functools
import struct
from typing import Sequence

import numpy as np

import torch

from cacheblend import _native as N
from cacheblend._timing import TIMES

_DT = {torch.bfloat16: N.CBK_BF16, torch.float16: N.CBK_F16}
ROPE_MODES = {"ref": N.CBK_ROPE_REF, "fp32": N.CBK_ROPE_FP32}


def _vp(x) -> ctypes.c_void_p:
    if x is None:
        return ctypes.c_void_p(0)
    return ctypes.c_void_p(x.data_ptr() if isinstance(x, torch.Tensor) else int(x))


def _stream(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def dtype_code(dt: torch.dtype) -> int:
    if dt not in _DT:
        raise NotImplementedError(f"libcbk kernels support bfloat16/float16 tensors, got {dt}")
    return _DT[dt]


def require_cuda(*ts: torch.Tensor) -> torch.device:
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("cacheblend kernels need CUDA tensors (no CPU path); got a "
                               f"{t.device} tensor")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"tensors on different devices: {dev} and {t.device}")
    return dev


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """Flatten to 2-D rows with unit inner stride and 16-byte aligned rows."""
    t2 = t.reshape(-1, t.shape[-1])
    if t2.stride(-1) != 1 or t2.stride(0) % 8 or t2.data_ptr() % 16:
        t2 = t2.contiguous()
    return t2


# ---------------------------------------------------------------------------
# RoPE
# ---------------------------------------------------------------------------
def rope_table(inv_freq: torch.Tensor, n_pos: int, scaling: float = 1.0) -> torch.Tensor:
    """(n_pos, D/2, 2) fp32 cos/sin table for positions 0..n_pos-1."""
    dev = require_cuda(inv_freq)
    inv = inv_freq.to(device=dev, dtype=torch.float32).contiguous()
    half = inv.numel()
    table = torch.empty((int(n_pos), half, 2), dtype=torch.float32, device=dev)
    with TIMES.span("rope_table", dev):
        N.check(N.LIB.cbk_rope_table(_vp(inv), half, int(n_pos), float(scaling), _vp(table), _stream(dev)),
              "cbk_rope_table")
    return table


def rope_rows(x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, head_dim: int,
              mode: str = "ref", out: torch.Tensor | None = None, status=None) -> torch.Tensor:
    """out[r] = RoPE(x[r], positions[r]) for rows of n_heads*head_dim elements."""
    dev = require_cuda(x, positions, table)
    xr = _rows(x, "x")
    pos = positions.reshape(-1).to(device=dev, dtype=torch.int64).contiguous()
    if pos.numel() != xr.shape[0]:
        raise ValueError(f"positions ({pos.numel()}) must match rows ({xr.shape[0]})")
    if out is None:
        out = torch.empty_like(xr)
    n_heads = xr.shape[1] // head_dim
    if n_heads * head_dim != xr.shape[1]:
        raise ValueError(f"row width {xr.shape[1]} is not a multiple of head_dim {head_dim}")
    with TIMES.span("rope_rows", dev):
        N.check(N.LIB.cbk_rope_rows(_vp(xr), _vp(out), xr.shape[0], n_heads, head_dim,
                                  dtype_code(x.dtype), _vp(table), table.shape[0], _vp(pos),
                                  ROPE_MODES[mode], _vp(status), _stream(dev)), "cbk_rope_rows")
    return out.view(x.shape)


# ---------------------------------------------------------------------------
# chunk tables
# ---------------------------------------------------------------------------
class ChunkTable:
    """Device descriptor table of chunk tensors: [layer][chunk] -> (K ptr, V ptr),
    plus the chunk start offsets (n_chunks + 1) in the fused sequence.

    Holds references to the chunk tensors so they outlive the kernels."""

    def __init__(self, entries: Sequence[dict], layers: Sequence[int], device: torch.device):
        self.n_chunks = len(entries)
        self.layers = list(layers)
        lens = []
        self._keep = []
        host = torch.empty((len(self.layers), self.n_chunks, 2), dtype=torch.int64, pin_memory=True)
        hv = host.numpy()
        kv_dim = None
        slabs = [e.get("_slab") for e in entries]
        if self.n_chunks and all(sl is not None for sl in slabs) and \
                len({(sl[0], sl[3], sl[4], sl[5]) for sl in slabs}) == 1:
            # chunks of one KVArena: the table follows from the slab offsets
            pool, _, _, row_elems, n_layers, kv_dim = slabs[0]
            t0 = entries[0]["K"][self.layers[0]]
            if t0.device != device:
                raise RuntimeError(f"chunk tensor on {t0.device}, model on {device}")
            esz = t0.element_size()
            first = np.array([sl[1] for sl in slabs], dtype=np.int64)
            lens_a = np.array([sl[2] for sl in slabs], dtype=np.int64)
            lay = np.array(self.layers, dtype=np.int64)
            if lay.min() < 0 or lay.max() >= n_layers:
                raise ValueError("chunk table layer out of range of the arena")
            kptr = pool + (first * row_elems)[None, :] * esz + lay[:, None] * (2 * lens_a * kv_dim * esz)[None, :]
            hv[:, :, 0] = kptr
            hv[:, :, 1] = kptr + (lens_a * kv_dim * esz)[None, :]
            lens = lens_a.tolist()
            self._keep = [e["K"][self.layers[0]] for e in entries]   # views keep the pool alive
            self._finish(host, lens, kv_dim, t0.dtype, device)
            return
        for c, e in enumerate(entries):
            for li, l in enumerate(self.layers):
                k = _chunk_rows(e["K"][l], device)
                v = _chunk_rows(e["V"][l], device)
                if k.shape != v.shape:
                    raise ValueError("chunk K and V shapes differ")
                if kv_dim is None:
                    kv_dim = k.shape[1]
                if k.shape[1] != kv_dim:
                    raise ValueError("chunk tensors have different widths")
                self._keep += [k, v]
                hv[li, c, 0] = k.data_ptr()
                hv[li, c, 1] = v.data_ptr()
                if li == 0:
                    lens.append(k.shape[0])
                elif k.shape[0] != lens[c]:
                    raise ValueError("chunk length differs across layers")
        self._finish(host, lens, kv_dim, self._keep[0].dtype, device)

    def _finish(self, host, lens, kv_dim, dtype, device):
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        hs = torch.tensor(starts, dtype=torch.int64).pin_memory()
        self.kv_dim = kv_dim
        self.S = starts[-1]
        self.lengths = lens
        self.srcs = host.to(device, non_blocking=True)
        self.starts = hs.to(device, non_blocking=True)
        self.dtype = dtype

    def refresh(self, entries: Sequence[dict]) -> None:
        """Point the same device table at other chunks of the same lengths
        (a captured graph reads it in place); ordered on the current stream."""
        new = ChunkTable(entries, self.layers, self.srcs.device)
        if new.lengths != self.lengths or new.kv_dim != self.kv_dim or new.dtype != self.dtype:
            raise ValueError("ChunkTable.refresh: chunk lengths / width / dtype differ from the table's")
        self.srcs.copy_(new.srcs, non_blocking=True)
        self._keep = new._keep

    def layer_ptr(self, layer: int) -> int:
        """Device address of the srcs row of one layer (n_chunks entries)."""
        li = self.layers.index(layer)
        return self.srcs.data_ptr() + li * self.n_chunks * 16


def chunk_signature(entries: Sequence[dict], layers: Sequence[int]) -> tuple:
    """Device addresses of the store entries' K/V tensors of `layers` (for
    KVArena entries, their slab): equal signatures mean a ChunkTable built from
    either set of entries holds the same pointers.  (A table keeps its tensors
    alive, so a stored tensor that replaced one of them cannot have its address.)"""
    sig = []
    for e in entries:
        slab = e.get("_slab")
        if slab is not None:
            sig.append(slab)
        else:
            K, V = e["K"], e["V"]
            sig.append(tuple(K[l].data_ptr() for l in layers) + tuple(V[l].data_ptr() for l in layers))
    return tuple(sig)


def _chunk_rows(t: torch.Tensor, device) -> torch.Tensor:
    if t.device != device:
        raise RuntimeError(f"chunk tensor on {t.device}, model on {device}")
    t2 = t.reshape(-1, t.shape[-1])
    if not t2.is_contiguous() or t2.data_ptr() % 16:
        t2 = t2.contiguous()
    return t2


# ---------------------------------------------------------------------------
# (a)+(b) assemble, (b)+(d) fresh-row scatter
# ---------------------------------------------------------------------------
def assemble_kv(table: ChunkTable, layer_lo: int, layer_hi: int, n_kv_heads: int, head_dim: int,
                rope: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor, mode: str = "ref",
                positions: torch.Tensor | None = None, status=None) -> None:
    """Fill k_out[l], v_out[l] (l in [layer_lo, layer_hi)) of [L][S][kv_dim]
    buffers from the chunk tensors, K rotated to its fused positions."""
    dev = require_cuda(k_out, v_out, rope)
    n_layers = layer_hi - layer_lo
    if n_layers <= 0:
        return
    li0 = table.layers.index(layer_lo)
    if table.layers[li0:li0 + n_layers] != list(range(layer_lo, layer_hi)):
        raise ValueError("chunk table does not hold the requested consecutive layers")
    srcs = table.srcs.data_ptr() + li0 * table.n_chunks * 16
    lstride = k_out.stride(0)
    kb = k_out.data_ptr() + layer_lo * lstride * k_out.element_size()
    vb = v_out.data_ptr() + layer_lo * lstride * v_out.element_size()
    with TIMES.span("assemble_kv", dev):
        N.check(N.LIB.cbk_assemble_kv(_vp(srcs), _vp(table.starts), table.n_chunks, n_layers, table.S,
                                    n_kv_heads, head_dim, dtype_code(k_out.dtype), _vp(rope),
                                    rope.shape[0], _vp(positions), ROPE_MODES[mode], _vp(kb), _vp(vb),
                                    lstride, _vp(status), _stream(dev)), "cbk_assemble_kv")


def rope_scatter(q_src: torch.Tensor, k_src: torch.Tensor, v_src: torch.Tensor, idx: torch.Tensor,
                 gather: bool, S: int, n_q_heads: int, n_kv_heads: int, head_dim: int,
                 rope: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 q_out: torch.Tensor | None = None, mode: str = "ref", status=None,
                 table_by_row: bool = False) -> torch.Tensor:
    """RoPE of fresh Q (-> q_out, [n_sel][Hq*D]) and K at positions idx; K and V
    rows written into the fused cache of one layer at rows idx.  With
    ``table_by_row`` row j of ``rope`` holds the cos/sin of position idx[j]
    (``rope.index_select(0, idx)``, made once per selection)."""
    dev = require_cuda(q_src, k_src, v_src, idx, rope, k_cache, v_cache)
    q2, k2, v2 = _rows(q_src, "q"), _rows(k_src, "k"), _rows(v_src, "v")
    n_sel = idx.numel()
    if q_out is None:
        q_out = torch.empty((n_sel, n_q_heads * head_dim), dtype=q_src.dtype, device=dev)
    with TIMES.span("rope_scatter", dev):
        N.check(N.LIB.cbk_rope_scatter(_vp(q2), q2.stride(0), _vp(k2), k2.stride(0), _vp(v2), v2.stride(0),
                                     int(bool(gather)), _vp(idx), n_sel, int(S), n_q_heads, n_kv_heads,
                                     head_dim, dtype_code(q_src.dtype), _vp(rope), rope.shape[0],
                                     ROPE_MODES[mode] | (N.CBK_ROPE_TABLE_BY_ROW if table_by_row else 0),
                                     _vp(q_out), _vp(k_cache), _vp(v_cache),
                                     _vp(status), _stream(dev)), "cbk_rope_scatter")
    return q_out


# ---------------------------------------------------------------------------
# (c) HKVD
# ---------------------------------------------------------------------------
def kv_deviation_rows(k_new: torch.Tensor, table: ChunkTable, layer: int) -> torch.Tensor:
    dev = require_cuda(k_new)
    kn = _rows(k_new, "K_new")
    out = torch.empty((table.S,), dtype=torch.float32, device=dev)
    with TIMES.span("kv_deviation", dev):
        N.check(N.LIB.cbk_kv_deviation(_vp(kn), kn.stride(0), _vp(table.layer_ptr(layer)),
                                     _vp(table.starts), table.n_chunks, table.S, kn.shape[1],
                                     dtype_code(k_new.dtype), _vp(out), _stream(dev)),
              "cbk_kv_deviation")
    return out


def topk_count(S: int, ratio: float) -> int:
    return int(N.LIB.cbk_topk_count(int(S), float(ratio)))


def topk_select(dev_scores: torch.Tensor, k: int, force_last: bool = False, status=None) -> torch.Tensor:
    dev = require_cuda(dev_scores)
    if dev_scores.dtype != torch.float32:
        dev_scores = dev_scores.float()
    d = dev_scores.contiguous()
    idx = torch.empty((int(k),), dtype=torch.int64, device=dev)
    with TIMES.span("topk_select", dev):
        N.check(N.LIB.cbk_topk_select(_vp(d), d.numel(), int(k), int(bool(force_last)), _vp(idx),
                                    _vp(status), _stream(dev)), "cbk_topk_select")
    return idx


def hkvd_select(k_new: torch.Tensor, table: ChunkTable, layer: int, k: int, force_last: bool = True,
                workspace: torch.Tensor | None = None, status=None):
    """Deviation of fresh K against the cached chunk K of `layer`, then top-K.
    Returns (indices, deviations) -- deviations live in the workspace."""
    dev = require_cuda(k_new)
    kn = _rows(k_new, "K_new")
    S = table.S
    need = int(N.LIB.cbk_hkvd_workspace_bytes(S))
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty((need // 4,), dtype=torch.float32, device=dev)
    idx = torch.empty((int(k),), dtype=torch.int64, device=dev)
    with TIMES.span("hkvd_select", dev, 2):
        N.check(N.LIB.cbk_hkvd_select(_vp(kn), kn.stride(0), _vp(table.layer_ptr(layer)),
                                    _vp(table.starts), table.n_chunks, S, kn.shape[1],
                                    dtype_code(k_new.dtype), int(k), int(bool(force_last)), _vp(idx),
                                    _vp(workspace), need, _vp(status), _stream(dev)),
              "cbk_hkvd_select")
    return idx, workspace.view(torch.float32)[:S]


# ---------------------------------------------------------------------------
# (e) partial attention
# ---------------------------------------------------------------------------
def attn_workspace(n_sel: int, S: int, n_q_heads: int, n_kv_heads: int, head_dim: int,
                   device) -> torch.Tensor:
    """Workspace for partial_attn (work plan + split partial results)."""
    nbytes = int(N.LIB.cbk_partial_attn_workspace_bytes(int(n_sel), int(S), n_q_heads, n_kv_heads, head_dim))
    if nbytes == 0:
        N.check(N.CBK_ERR_INVALID, "cbk_partial_attn_workspace_bytes")
    return torch.empty((nbytes,), dtype=torch.uint8, device=device)


def partial_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: torch.Tensor,
                 n_q_heads: int, n_kv_heads: int, head_dim: int, scale: float,
                 out: torch.Tensor | None = None, status=None, workspace: torch.Tensor | None = None,
                 reuse_plan: bool = False, timer_tag: str = "") -> torch.Tensor:
    """softmax(scale q k^T, keys <= pos) v for selected rows.

    q: [n_sel][Hq*D] (rotated); k_cache/v_cache: [S][Hkv*D]; pos: int64 [n_sel]
    ascending.  Returns [n_sel][Hq*D].  ``workspace`` (from attn_workspace) may
    be shared by calls with the same pos; ``reuse_plan`` skips re-planning."""
    dev = require_cuda(q, k_cache, v_cache, pos)
    n_sel = pos.numel()
    S = k_cache.shape[0]
    for t, name in ((q, "q"), (k_cache, "k_cache"), (v_cache, "v_cache")):
        if not t.is_contiguous():
            raise ValueError(f"partial_attn: {name} must be contiguous")
    if out is None:
        out = torch.empty((n_sel, n_q_heads * head_dim), dtype=q.dtype, device=dev)
    if workspace is None:
        workspace = attn_workspace(n_sel, S, n_q_heads, n_kv_heads, head_dim, dev)
        reuse_plan = False
    with TIMES.span("partial_attn" + timer_tag, dev, 2 if reuse_plan else 3):   # plan, attention, combine
        N.check(N.LIB.cbk_partial_attn(_vp(q), _vp(k_cache), _vp(v_cache), _vp(pos), n_sel, S,
                                       n_q_heads, n_kv_heads, head_dim, float(scale),
                                       dtype_code(q.dtype), _vp(out), _vp(workspace), workspace.numel(),
                                       int(bool(reuse_plan)), _vp(status), _stream(dev)),
                "cbk_partial_attn")
    return out


# ---------------------------------------------------------------------------
# decoder-layer row kernels (RMSNorm with residual add, SiLU * up)
# ---------------------------------------------------------------------------
def add_rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, delta: torch.Tensor | None = None,
                rows: torch.Tensor | None = None, sum_out: torch.Tensor | None = None,
                out: torch.Tensor | None = None, status=None) -> torch.Tensor:
    """HF RMSNorm of ``s`` = x (rows gathered by ``rows`` when given) plus ``delta``
    (16-bit residual add), in one pass.  ``s`` is written to ``sum_out`` when
    given (it may be ``x`` itself when ``rows`` is None).  x: [..., cols]; the
    result has delta's / the gathered row count and x's last dimension."""
    dev = require_cuda(x, weight, delta, rows, sum_out, out)
    x2 = _rows(x, "x")
    cols = x2.shape[1]
    if weight.dtype != x.dtype or weight.numel() != cols:
        raise ValueError(f"add_rmsnorm: weight must be {x.dtype}[{cols}], got {weight.dtype}{list(weight.shape)}")
    w = weight.contiguous()
    if rows is not None:
        if rows.dtype != torch.int64:
            raise ValueError("add_rmsnorm: rows must be int64")
        rows = rows.contiguous()
        n = rows.numel()
    else:
        n = x2.shape[0]
    d2 = None
    if delta is not None:
        if delta.dtype != x.dtype or delta.shape[-1] != cols or delta.numel() != n * cols:
            raise ValueError(f"add_rmsnorm: delta must be {x.dtype} with {n} rows of {cols}")
        d2 = _rows(delta, "delta")
    lead = (delta.shape[:-1] if delta is not None else
            (x.shape[:-1] if rows is None else (1, n) if x.dim() == 3 else (n,)))
    if out is None:
        out = torch.empty((*lead, cols), dtype=x.dtype, device=dev)
    o2 = out.view(-1, cols)
    s2 = None
    if sum_out is not None:
        if sum_out.dtype != x.dtype or sum_out.numel() != n * cols:
            raise ValueError(f"add_rmsnorm: sum_out must be {x.dtype} with {n} rows of {cols}")
        if rows is not None and sum_out.data_ptr() == x2.data_ptr():
            raise ValueError("add_rmsnorm: sum_out may alias x only without a row gather")
        s2 = sum_out.view(-1, cols)
    with TIMES.span("add_rmsnorm", dev):
        N.check(N.LIB.cbk_add_rmsnorm(_vp(x2), x2.stride(0), x2.shape[0], _vp(rows), _vp(d2),
                                      d2.stride(0) if d2 is not None else 0, _vp(s2),
                                      s2.stride(0) if s2 is not None else 0, _vp(w), float(eps), n, cols,
                                      dtype_code(x.dtype), _vp(o2), o2.stride(0), _vp(status), _stream(dev)),
                "cbk_add_rmsnorm")
    return out


def silu_mul(gate: torch.Tensor, up: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """round16(silu(gate)) * up with the 16-bit roundings of torch's SiLU and mul."""
    dev = require_cuda(gate, up, out)
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise ValueError(f"silu_mul: gate {gate.dtype}{list(gate.shape)} vs up {up.dtype}{list(up.shape)}")
    g2, u2 = _rows(gate, "gate"), _rows(up, "up")
    if out is None:
        out = torch.empty(gate.shape, dtype=gate.dtype, device=dev)
    o2 = out.view(-1, gate.shape[-1])
    with TIMES.span("silu_mul", dev):
        N.check(N.LIB.cbk_silu_mul(_vp(g2), g2.stride(0), _vp(u2), u2.stride(0), g2.shape[0], g2.shape[1],
                                   dtype_code(gate.dtype), _vp(o2), o2.stride(0), _stream(dev)),
                "cbk_silu_mul")
    return out


def gemv(weight: torch.Tensor, x: torch.Tensor | None = None, gate: torch.Tensor | None = None,
         up: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """One-row projection x @ weight.T (a decode step's Linear), fp32 accumulation,
    shape (..., N) for x of shape (..., K) with one row.  With gate and up instead
    of x, the input is round16(round16(silu(gate)) * up) (silu_mul's arithmetic)."""
    src = x if x is not None else gate
    dev = require_cuda(weight, src, up, out)
    if (x is None) == (gate is None) or (gate is None) != (up is None):
        raise ValueError("gemv: pass x, or gate and up")
    k = weight.shape[1]
    if src.shape[-1] != k or src.numel() != k or (up is not None and up.shape != gate.shape):
        raise ValueError(f"gemv: one input row of {k} elements expected, got {list(src.shape)}")
    if weight.stride(1) != 1:
        raise ValueError("gemv: weight rows must be contiguous")
    if out is None:
        out = torch.empty((*src.shape[:-1], weight.shape[0]), dtype=weight.dtype, device=dev)
    xs = [t if t is None or t.is_contiguous() else t.contiguous() for t in (x, gate, up)]
    with TIMES.span("gemv", dev):
        N.check(N.LIB.cbk_gemv(_vp(weight), weight.stride(0), _vp(xs[0]), _vp(xs[1]), _vp(xs[2]), weight.shape[0],
                               k, dtype_code(weight.dtype), _vp(out), _stream(dev)), "cbk_gemv")
    return out


def decode_workspace(cap: int, n_q_heads: int, n_kv_heads: int, head_dim: int, device) -> torch.Tensor:
    """Workspace of decode_attn for a cache of `cap` rows (per-split partial
    results; reusable by calls that do not overlap on the GPU)."""
    n = N.LIB.cbk_decode_attn_workspace_bytes(int(cap), n_q_heads, n_kv_heads, head_dim)
    if n == 0:
        raise ValueError("decode_workspace: bad geometry")
    return torch.zeros((n,), dtype=torch.uint8, device=device)


def decode_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: torch.Tensor,
                n_q_heads: int, n_kv_heads: int, head_dim: int, scale: float, workspace: torch.Tensor,
                out: torch.Tensor | None = None, status=None) -> torch.Tensor:
    """Attention of one query token (q: [n_q_heads * head_dim], rotated) at the
    device position pos (int64, one element) over cache rows 0..pos of
    k_cache / v_cache ([cap][n_kv_heads * head_dim]); returns [1][n_q_heads * head_dim]."""
    dev = require_cuda(q, k_cache, v_cache, pos, workspace)
    if pos.dtype != torch.int64 or pos.numel() != 1:
        raise ValueError("decode_attn: pos must be one int64 on the device")
    if k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride() or k_cache.stride(-1) != 1:
        raise ValueError("decode_attn: k_cache and v_cache must have the same row layout")
    qc = q.reshape(-1)
    if not qc.is_contiguous():
        qc = qc.contiguous()
    if out is None:
        out = torch.empty((1, n_q_heads * head_dim), dtype=q.dtype, device=dev)
    with TIMES.span("decode_attn", dev):
        N.check(N.LIB.cbk_decode_attn(_vp(qc), _vp(k_cache), _vp(v_cache), k_cache.stride(0), _vp(pos),
                                      k_cache.shape[0], n_q_heads, n_kv_heads, head_dim, float(scale),
                                      dtype_code(q.dtype), _vp(out), _vp(workspace), workspace.numel(),
                                      _vp(status), _stream(dev)), "cbk_decode_attn")
    return out


def scatter_rows(src: torch.Tensor, idx: torch.Tensor, n_rows: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """Dense [n_rows][...] rows: out[idx[j]] = src[j], zeros elsewhere (idx ascending,
    distinct), every output byte written once."""
    dev = require_cuda(src, idx, out)
    s2 = _rows(src, "src")
    if idx.dtype != torch.int64 or idx.numel() != s2.shape[0]:
        raise ValueError("scatter_rows: idx must be int64 with one entry per source row")
    idx = idx.contiguous()
    if out is None:
        out = torch.empty((n_rows, s2.shape[1]), dtype=src.dtype, device=dev)
    o2 = out.view(-1, s2.shape[1])
    if o2.shape[0] != n_rows:
        raise ValueError(f"scatter_rows: out has {o2.shape[0]} rows, expected {n_rows}")
    row_bytes = s2.shape[1] * s2.element_size()
    with TIMES.span("scatter_rows", dev):
        N.check(N.LIB.cbk_scatter_rows(_vp(s2), s2.stride(0) * s2.element_size(), _vp(idx), idx.numel(), _vp(o2),
                                       o2.stride(0) * o2.element_size(), int(n_rows), row_bytes, _stream(dev)),
                "cbk_scatter_rows")
    return out


# ---------------------------------------------------------------------------
# decoding with drafted tokens
# ---------------------------------------------------------------------------
_DT3 = {**_DT, torch.float32: N.CBK_F32}


def _launcher(name: str, n_launches: int):
    """Caller of one C-ABI entry that takes a packed argument struct: on dev's
    current stream, with dev the current device meanwhile and the span timed when
    timing is on.  (What it needs is looked up once: these calls are short enough
    for the lookups to show.)"""
    entry = "cbk_" + name
    fmt = N.PACK[entry]
    pack, size, fn = fmt.pack, fmt.size, getattr(N.LIB, entry)
    raw_stream, current_device = torch._C._cuda_getCurrentRawStream, torch.cuda.current_device

    def launch(dev: torch.device, *args) -> None:
        index = dev.index
        try:
            packed = pack(size, *args)
        except (OverflowError, struct.error) as e:
            raise ValueError(f"{entry}: an argument does not fit its field ({e})") from None
        if TIMES.active or current_device() != index:
            with torch.cuda.device(dev), TIMES.span(name, dev, n_launches):
                rc = fn(packed, raw_stream(index))
        else:
            rc = fn(packed, raw_stream(index))
        if rc:
            N.check(rc, entry)
    return launch


_norm_rope_scatter = _launcher("norm_rope_scatter", 1)
_tree_attn = _launcher("tree_attn", 2)
_process_logits = _launcher("process_logits", 2)


def _same_device(first: torch.Tensor, *others) -> torch.device:
    """require_cuda for calls where its cost shows: the device all tensors are on."""
    at = first.get_device()
    for t in others:
        if t is not None and t.get_device() != at:
            at = -1
    if at < 0:
        require_cuda(first, *others)
    return first.device


def _src_rows(t: torch.Tensor, n: int, cols: int, who: str) -> tuple[torch.Tensor, int]:
    """(t as n rows of cols elements, row stride), in place where its rows can be read as they are."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.shape != (n, cols):
        raise ValueError(f"{who} must be {n} rows of {cols}, got {list(t.shape)}")
    row, col = t.stride()
    if col != 1 or row % 8 or row < cols or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        row = cols
    return t, row


def _index(t: torch.Tensor, n: int, who: str) -> torch.Tensor:
    if t.dtype != torch.int64 or t.numel() != n:
        raise ValueError(f"{who} must be int64 with {n} entries, got {t.dtype}{list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, dtype, kv_dim: int, who: str) -> tuple[int, int]:
    """(rows, row stride) of the caches."""
    if k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise ValueError(f"{who}: caches must be {dtype}, got {k_cache.dtype} / {v_cache.dtype}")
    shape, stride = k_cache.shape, k_cache.stride()
    if len(shape) != 2 or shape != v_cache.shape or stride != v_cache.stride() or shape[1] != kv_dim or stride[1] != 1:
        raise ValueError(f"{who}: k_cache and v_cache must be rows of {kv_dim} elements with one layout, got "
                         f"{list(shape)} and {list(v_cache.shape)}")
    return shape[0], stride[0]


def norm_rope_scatter(q_src: torch.Tensor, k_src: torch.Tensor, v_src: torch.Tensor, positions: torch.Tensor,
                      rows: torch.Tensor, n_q_heads: int, n_kv_heads: int, head_dim: int, rope: torch.Tensor,
                      k_cache: torch.Tensor, v_cache: torch.Tensor, q_weight: torch.Tensor | None = None,
                      k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False,
                      q_out: torch.Tensor | None = None, mode: str = "ref", status=None) -> torch.Tensor:
    """Per-head RMSNorm (with ``q_weight`` and ``k_weight``) and rotation of Q and K
    at ``positions``; K and V into cache rows ``rows``.  Returns the rotated Q,
    [n][Hq*D].

    q_src / k_src / v_src: n rows of heads (views of one stacked projection are
    read in place; q_out and the caches must not overlap them); ``positions`` and
    ``rows``: int64, n entries -- siblings of a drafted tree share a position, not a
    row; rows are distinct, and a row of -1 marks a padding token of which nothing is
    written.  ``rope``: fp32 (cos, sin)
    table [n_pos][R / 2][2]; the first R dimensions of a head are rotated, as the
    pairs (i, i + R / 2) or, ``interleaved``, (2i, 2i + 1).  k_cache / v_cache:
    [cap][Hkv*D].  ``mode`` "ref" rounds to 16 bits where the HF modules do, "fp32"
    once.  A position or row outside its buffer sets CBK_STATUS_BAD_INDEX and
    skips the token."""
    dev = _same_device(q_src, k_src, v_src, positions, rows, rope, k_cache, v_cache, q_weight, k_weight, q_out,
                       status)
    dt = q_src.dtype
    code = _DT.get(dt)
    if code is None:
        dtype_code(dt)
    if mode not in ROPE_MODES:
        raise ValueError(f"norm_rope_scatter: mode must be one of {sorted(ROPE_MODES)}, got {mode!r}")
    if k_src.dtype != dt or v_src.dtype != dt:
        raise ValueError(f"norm_rope_scatter: q, k and v must have one dtype, got {dt}, {k_src.dtype}, {v_src.dtype}")
    n, qd, kd = rows.numel(), n_q_heads * head_dim, n_kv_heads * head_dim
    q2, qs = _src_rows(q_src, n, qd, "norm_rope_scatter: q_src")
    k2, ks = _src_rows(k_src, n, kd, "norm_rope_scatter: k_src")
    v2, vs = _src_rows(v_src, n, kd, "norm_rope_scatter: v_src")
    positions = _index(positions, n, "norm_rope_scatter: positions")
    rows = _index(rows, n, "norm_rope_scatter: rows")
    table = rope.shape
    if rope.dtype != torch.float32 or len(table) != 3 or table[2] != 2 or not rope.is_contiguous():
        raise ValueError("norm_rope_scatter: rope must be a contiguous fp32 table [n_pos][R / 2][2]")
    cap, kvs = _check_cache(k_cache, v_cache, dt, kd, "norm_rope_scatter")
    qw = kw = 0
    if q_weight is not None and k_weight is not None:
        for w in (q_weight, k_weight):
            if w.dtype != dt or w.numel() != head_dim or not w.is_contiguous():
                raise ValueError(f"norm_rope_scatter: weights must be contiguous {dt}[{head_dim}], got "
                                 f"{w.dtype}{list(w.shape)}")
        qw, kw = q_weight.data_ptr(), k_weight.data_ptr()
    elif q_weight is not None or k_weight is not None:
        raise ValueError("norm_rope_scatter: give both q_weight and k_weight, or neither")
    if q_out is None:
        q_out = torch.empty_like(q2, memory_format=torch.contiguous_format)
    elif q_out.dtype != dt or q_out.numel() != n * qd or not q_out.is_contiguous():
        raise ValueError(f"norm_rope_scatter: q_out must be contiguous {dt} with {n} rows of {qd}")
    _norm_rope_scatter(dev, q2.data_ptr(), k2.data_ptr(), v2.data_ptr(), positions.data_ptr(), rows.data_ptr(), qw, kw,
                       rope.data_ptr(), q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                       0 if status is None else status.data_ptr(), qs, ks, vs, kvs, n, table[0], cap, n_q_heads,
                       n_kv_heads, head_dim, 2 * table[1], bool(interleaved), code, ROPE_MODES[mode], eps)
    return q_out


@functools.lru_cache(maxsize=1024)
def _tree_workspace_bytes(n_nodes: int, cap: int, n_q_heads: int, n_kv_heads: int, head_dim: int, index: int) -> int:
    """Workspace size on device ``index`` (it goes by that device's SMs)."""
    if head_dim not in (64, 128) or n_nodes > 1024:
        raise NotImplementedError(f"tree_attn: head_dim 64 or 128 and at most 1024 nodes, got {head_dim}, {n_nodes}")
    with torch.cuda.device(index):
        nbytes = N.LIB.cbk_tree_attn_workspace_bytes(n_nodes, cap, n_q_heads, n_kv_heads, head_dim)
    if nbytes == 0:
        raise ValueError(f"tree_workspace: {N.last_error()}")
    return nbytes


def tree_workspace(n_nodes: int, cap: int, n_q_heads: int, n_kv_heads: int, head_dim: int, device) -> torch.Tensor:
    """Workspace of tree_attn for n_nodes nodes over a cache of cap rows (reusable by
    calls that do not overlap on the GPU; another number of nodes may need more)."""
    device = torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    nbytes = _tree_workspace_bytes(n_nodes, cap, n_q_heads, n_kv_heads, head_dim, index)
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def tree_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, n_ctx: torch.Tensor,
              words: torch.Tensor, n_q_heads: int, n_kv_heads: int, head_dim: int, scale: float,
              workspace: torch.Tensor | None = None, out: torch.Tensor | None = None, status=None) -> torch.Tensor:
    """Attention of a tree of T drafted tokens over cache rows [0, n_ctx) and the
    nodes' own rows n_ctx + j, of which node i sees those with bit j of
    ``words[i]`` set (int32 [T][>= ceil(T / 32)], bit j % 32 of word j / 32; see
    ``tree_words``).  q: [T][Hq*D] (rotated); ``n_ctx``: one int64 on the device,
    so that a captured step stays valid as it advances; returns [T][Hq*D].  A
    node that sees no row gets zeros; masked rows and rows behind the tree may
    hold anything.  n_ctx + T beyond the cache sets CBK_STATUS_BAD_INDEX and
    leaves ``out`` as it was."""
    dev = _same_device(q, k_cache, v_cache, n_ctx, words, workspace, out, status)
    dt = q.dtype
    code = _DT.get(dt)
    if code is None:
        dtype_code(dt)
    ws, qd = words.shape, n_q_heads * head_dim
    if words.dtype != torch.int32 or len(ws) != 2 or ws[1] * 32 < ws[0] or words.stride(1) != 1:
        raise ValueError(f"tree_attn: words must be int32 [T][>= ceil(T / 32)] rows, got {words.dtype}{list(ws)}")
    t = ws[0]
    if q.numel() != t * qd or q.shape[-1] != qd:
        raise ValueError(f"tree_attn: q must be {t} rows of {qd}, got {list(q.shape)}")
    if n_ctx.dtype != torch.int64 or n_ctx.numel() != 1:
        raise ValueError("tree_attn: n_ctx must be one int64 on the device")
    cap, kvs = _check_cache(k_cache, v_cache, dt, n_kv_heads * head_dim, "tree_attn")
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    words, words_stride = _word_rows(words)
    if workspace is None:
        workspace = torch.empty(_tree_workspace_bytes(t, cap, n_q_heads, n_kv_heads, head_dim, dev.index),
                                dtype=torch.uint8, device=dev)
    elif workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise ValueError("tree_attn: workspace must come from tree_workspace")
    if out is None:
        out = torch.empty_like(q) if q.dim() == 2 else torch.empty_like(q).view(t, qd)
    elif out.dtype != dt or out.numel() != t * qd or not out.is_contiguous():
        raise ValueError(f"tree_attn: out must be contiguous {dt} with {t} rows of {qd}")
    _tree_attn(dev, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), n_ctx.data_ptr(), words.data_ptr(),
               out.data_ptr(), workspace.data_ptr(), 0 if status is None else status.data_ptr(), kvs, words_stride,
               cap, workspace.numel(), t, n_q_heads, n_kv_heads, head_dim, code, scale)
    return out


def tree_words(parents: Sequence[int], width: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(words, depth) of a drafted tree given each node's parent (-1 for a root,
    else an earlier node): words int32 [T][width] (default ceil(T / 32)) with bit
    j of row i set for node i and its ancestors, depth int64 [T] (0 for a root);
    both on the host."""
    n = len(parents)
    need = max(1, (n + 31) // 32)
    width = need if width is None else width
    if width < need:
        raise ValueError(f"tree_words: {n} nodes need {need} words, got width {width}")
    seen = np.zeros((n, 32 * width), dtype=np.uint8)
    depth = np.zeros((n,), dtype=np.int64)
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            raise ValueError(f"tree_words: node {i} has parent {p} (-1 or an earlier node)")
        if p >= 0:
            seen[i] = seen[p]
            depth[i] = depth[p] + 1
        seen[i, i] = 1
    words = np.packbits(seen, axis=1, bitorder="little").view("<i4").astype(np.int32)
    return torch.from_numpy(words), torch.from_numpy(depth)


def mask_words(allowed: torch.Tensor) -> torch.Tensor:
    """int32 bit words (..., ceil(n / 32)) of a bool tensor (..., n), on its device:
    bit t % 32 of word t / 32 is entry t (process_logits' ``mask_words``)."""
    if allowed.dtype != torch.bool:
        raise ValueError(f"mask_words: bool tensor expected, got {allowed.dtype}")
    n = allowed.shape[-1]
    wide = torch.zeros((*allowed.shape[:-1], (n + 31) // 32 * 32), dtype=torch.int64, device=allowed.device)
    wide[..., :n] = allowed
    words = (wide.view(*allowed.shape[:-1], -1, 32) << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _word_rows(words: torch.Tensor) -> tuple[torch.Tensor, int]:
    """2-D bit words and their row stride; broadcast or overlapping rows are copied apart."""
    if words.shape[0] <= 1:
        return words, words.shape[1]
    if words.stride(0) < words.shape[1]:
        words = words.contiguous()
    return words, words.stride(0)


def _row_stride(t: torch.Tensor, rows: int, cols: int, who: str) -> tuple[torch.Tensor, int, int]:
    """t as [rows][>= cols] or one shared row: (tensor with unit inner stride, row length, row stride or 0)."""
    shape = t.shape
    if len(shape) == 1:
        shape = (1, shape[0])
    if len(shape) != 2 or (shape[0] != 1 and shape[0] != rows) or shape[1] < cols:
        raise ValueError(f"{who} must be one row or {rows} rows of at least {cols}, got {list(t.shape)}")
    stride = t.stride()
    if stride[-1] != 1 and shape[1] > 1:
        t = t.contiguous()
        stride = t.stride()
    return t, shape[1], (0 if shape[0] == 1 else stride[0])


def process_logits(logits: torch.Tensor, history: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                   n_prompt: torch.Tensor | None = None, repetition: float = 1.0, presence: float = 0.0,
                   frequency: float = 0.0, bias: torch.Tensor | None = None, mask_words: torch.Tensor | None = None,
                   tree_tokens: torch.Tensor | None = None, tree_words: torch.Tensor | None = None,
                   out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None, return_logits: bool = True,
                   status=None):
    """Penalties for repeated tokens, bias and grammar mask on rows of logits, and
    the token each row chooses: (processed logits or None, int64 tokens).

    logits: [rows][vocab] bf16, fp16 or fp32 (leading dimensions are kept).
    ``history``: int64 token ids, one row for all or one per row, of which the
    first ``lengths`` (int64 on the device, one or one per row; default all) count
    and the first ``n_prompt`` of those are the prompt's (default none); the rest
    were made.  With ``tree_tokens`` / ``tree_words`` row r is a node of a drafted
    tree and the tokens on its path were made too.  A token made c times or in
    the prompt: x / repetition if x > 0, else x * repetition; made: x - frequency *
    c - presence; then ``bias`` (fp32, one row or one per row) and, where
    ``mask_words`` (int32, bit t % 32 of word t / 32) has a clear bit, -inf.  The
    token is the first largest value (NaN counts as largest); a row of -inf
    chooses 0.  ``out`` may be ``logits``; ``out_dtype`` is the logits' (default)
    or fp32."""
    dev = _same_device(logits, history, lengths, n_prompt, bias, mask_words, tree_tokens, tree_words, out, status)
    dt = logits.dtype
    code = _DT3.get(dt)
    if code is None:
        raise NotImplementedError(f"process_logits: bf16, fp16 or fp32 logits, got {dt}")
    shape = logits.shape
    flat = len(shape) == 2
    if not flat:
        logits = logits.reshape(-1, shape[-1])
    rows, vocab = logits.shape
    row_stride, col = logits.stride()
    if col != 1 or (rows > 1 and row_stride < vocab):
        logits = logits.contiguous()
        row_stride = vocab
    hist = lens = prompt = bias_p = mask_p = toks = words = 0
    hist_stride = hist_cap = len_stride = prompt_stride = bias_stride = mask_stride = tree_stride = n_tree = 0
    if history is not None:
        if history.dtype != torch.int64:
            raise ValueError(f"process_logits: history must be int64, got {history.dtype}")
        history, hist_cap, hist_stride = _row_stride(history, rows, 0, "process_logits: history")
        hist = history.data_ptr()
        if lengths is not None:
            n = lengths.numel()
            lengths = _index(lengths, 1 if n == 1 else rows, "process_logits: lengths")
            lens, len_stride = lengths.data_ptr(), n != 1
        if n_prompt is not None:
            n = n_prompt.numel()
            n_prompt = _index(n_prompt, 1 if n == 1 else rows, "process_logits: n_prompt")
            prompt, prompt_stride = n_prompt.data_ptr(), n != 1
    elif lengths is not None or n_prompt is not None:
        raise ValueError("process_logits: lengths and n_prompt belong to a history")
    if tree_tokens is not None and tree_words is not None:
        n_tree = tree_tokens.numel()
        tree_tokens = _index(tree_tokens, n_tree, "process_logits: tree_tokens")
        ws = tree_words.shape
        if (tree_words.dtype != torch.int32 or len(ws) != 2 or ws[0] != rows or ws[1] * 32 < n_tree
                or tree_words.stride(1) != 1):
            raise ValueError(f"process_logits: tree_words must be int32, {rows} rows of at least {n_tree} bits")
        tree_words, tree_stride = _word_rows(tree_words)
        toks, words = tree_tokens.data_ptr(), tree_words.data_ptr()
    elif tree_tokens is not None or tree_words is not None:
        raise ValueError("process_logits: give both tree_tokens and tree_words, or neither")
    if bias is not None:
        if bias.dtype != torch.float32:
            raise ValueError(f"process_logits: bias must be fp32, got {bias.dtype}")
        bias, _, bias_stride = _row_stride(bias, rows, vocab, "process_logits: bias")
        bias_p = bias.data_ptr()
    if mask_words is not None:
        if mask_words.dtype != torch.int32:
            raise ValueError(f"process_logits: mask_words must be int32, got {mask_words.dtype}")
        mask_words, _, mask_stride = _row_stride(mask_words, rows, (vocab + 31) // 32, "process_logits: mask_words")
        mask_p = mask_words.data_ptr()
    out_p = out_code = out_stride = 0
    if out is not None:
        if out_dtype not in (None, out.dtype):
            raise ValueError(f"process_logits: out is {out.dtype}, out_dtype {out_dtype}")
        if out.numel() != rows * vocab or out.shape[-1] != vocab:
            raise ValueError(f"process_logits: out must be {rows} rows of {vocab}, got {list(out.shape)}")
        out2 = out.view(-1, vocab)
        out_stride, col = out2.stride()
        if col != 1:
            raise ValueError("process_logits: out rows must be contiguous")
        out_p, out_code = out2.data_ptr(), _DT3.get(out.dtype)
    elif return_logits:
        out = torch.empty_like(logits, dtype=out_dtype, memory_format=torch.contiguous_format)
        if not flat:
            out = out.view(shape)
        out_p, out_code, out_stride = out.data_ptr(), _DT3.get(out.dtype), vocab
    if out_code is None:
        raise NotImplementedError(f"process_logits: bf16, fp16 or fp32 output, got {out.dtype}")
    tokens = torch.empty(rows if flat else shape[:-1], dtype=torch.int64, device=dev)
    if not (0 < repetition < float("inf") and presence == presence and frequency == frequency):
        raise ValueError("process_logits: repetition must be positive and finite, and no penalty NaN")
    if repetition == 1.0 and presence == 0.0 and frequency == 0.0:
        hist_cap = n_tree = 0                    # nothing depends on the counts
    ws = ws_bytes = 0
    if hist_cap and rows > 1 and not (hist_stride or len_stride or prompt_stride):
        ws_bytes = N.LIB.cbk_process_logits_workspace_bytes(rows, vocab)
        if ws_bytes:
            workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
            ws = workspace.data_ptr()
    if rows == 1:                                # one row's stride says nothing
        row_stride = out_stride = vocab
    _process_logits(dev, logits.data_ptr(), hist, lens, prompt, bias_p, mask_p, toks, words, out_p, tokens.data_ptr(),
                    0 if status is None else status.data_ptr(), ws, row_stride, rows, vocab, hist_stride, hist_cap,
                    len_stride, prompt_stride, bias_stride, mask_stride, tree_stride, out_stride, ws_bytes, n_tree,
                    code, out_code, repetition, presence, frequency)
    return out, tokens
