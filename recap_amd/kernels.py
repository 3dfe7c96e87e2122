"""torch-facing wrappers of the HIP kernels: argument checks, output allocation, streams.

Every function runs on ``torch.cuda.current_stream()`` and allocates its outputs with the
caching allocator; the kernels themselves never allocate.  Tensors are passed to the C ABI
as raw device pointers with explicit strides.
"""

from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import call

BLOCK = 128


def dtype_code(dtype: torch.dtype) -> int:
    if dtype == torch.bfloat16:
        return _lib.RECAP_BF16
    if dtype == torch.float16:
        return _lib.RECAP_F16
    raise ValueError(f"unsupported attention dtype {dtype}; use bfloat16 or float16")


def _stream() -> int:
    """The current stream's handle (what torch.cuda.current_stream() wraps, 5 us faster)."""
    torch.cuda.init()
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _p(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


@dataclass(frozen=True)
class Geometry:
    """Block geometry of one sequence (recap/sparse/attention.py:42-52,
    recap/kernels/block_sparse.py:60-74)."""

    n_tokens: int
    n_video: int
    # Video blocks per closure-statistics workgroup, fixed for a whole layer (the partial
    # sums, and so the rounding, depend on it); None: chosen from the call's banks.
    closure_group: int | None = None
    # (group, parts) of the per-call statistics, fixed for a whole layer likewise.
    closure_span: tuple[int, int] | None = None
    # Segments of each long query row of the masked attention, fixed for a whole layer like
    # the group above; None: chosen from the call's banks.
    attn_split: int | None = None

    @property
    def nb(self) -> int:
        return (self.n_video + BLOCK - 1) // BLOCK

    @property
    def tb(self) -> int:
        return (self.n_tokens + BLOCK - 1) // BLOCK

    @property
    def ds(self) -> int:
        shared = self.n_video % BLOCK != 0 and self.n_tokens > self.n_video
        return self.nb - 1 if shared else self.nb

    @property
    def rows(self) -> int:
        return (self.n_video // BLOCK) * BLOCK

    @property
    def partial(self) -> bool:
        return self.n_video % BLOCK != 0

    def counts(self, device) -> torch.Tensor:
        c = torch.full((self.nb,), float(BLOCK), dtype=torch.float32, device=device)
        c[-1] = float(self.n_video - BLOCK * (self.nb - 1))
        return c


def prepare(x: torch.Tensor, name: str) -> torch.Tensor:
    """A ``[B, H, N, D]`` view the kernels can read: unit dim stride, strides and base
    pointer 16-byte aligned; otherwise a contiguous copy."""
    if x.ndim != 4:
        raise ValueError(f"{name} must be [batch, heads, tokens, dim], got {tuple(x.shape)}")
    if not x.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    dtype_code(x.dtype)
    if x.shape[-1] not in (64, 128):
        raise ValueError(f"{name}: head dim {x.shape[-1]} unsupported (64 or 128)")
    ok = (x.stride(-1) == 1 and all(s % 8 == 0 for s in x.stride()[:3])
          and x.data_ptr() % 16 == 0)
    if not ok:
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
    return x


def _same_type(q: torch.Tensor, kv: "PackedKV") -> None:
    """The kernels read Q and the packed K/V tiles in one element type."""
    if q.dtype != kv.dtype:
        raise ValueError(f"Q is {q.dtype} but the packed K/V tiles are {kv.dtype}")


def _qkv_args(x: torch.Tensor):
    b, h, _, d = x.shape
    return [x.data_ptr(), dtype_code(x.dtype), b, h, d, x.stride(0), x.stride(1), x.stride(2)]


# -- stage 1 -------------------------------------------------------------------------------


@dataclass
class PackedKV:
    """Packed K / V^T tiles and fp32 block means of one call."""

    k_tiles: torch.Tensor   # [banks, tb, 128*d] (K tile images)
    vt_tiles: torch.Tensor  # [banks, tb, 128*d] (V^T tile images)
    k_means: torch.Tensor   # [banks, nb, d] fp32
    v_means: torch.Tensor   # [banks, nb, d] fp32
    dtype: torch.dtype
    dim: int


def kv_pack(k: torch.Tensor, v: torch.Tensor, rowmap: torch.Tensor, geo: Geometry) -> PackedKV:
    if k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError("K and V must have the same shape and dtype")
    b, h, n, d = k.shape
    banks = b * h
    kt = torch.empty(banks, geo.tb, BLOCK * d, dtype=k.dtype, device=k.device)
    vt = torch.empty_like(kt)
    km = torch.empty(banks, geo.nb, d, dtype=torch.float32, device=k.device)
    vm = torch.empty_like(km)
    call("recap_kv_pack", k.data_ptr(), v.data_ptr(), dtype_code(k.dtype), b, h, d,
         k.stride(0), k.stride(1), k.stride(2), v.stride(0), v.stride(1), v.stride(2),
         rowmap.data_ptr(), n, geo.n_video, kt.data_ptr(), vt.data_ptr(), km.data_ptr(),
         vm.data_ptr(), _stream())
    return PackedKV(kt, vt, km, vm, k.dtype, d)


def pool_blocks(x: torch.Tensor, rowmap: torch.Tensor, geo: Geometry) -> torch.Tensor:
    b, h, n, d = x.shape
    out = torch.empty(b * h, geo.nb, d, dtype=torch.float32, device=x.device)
    call("recap_pool_blocks", *_qkv_args(x), rowmap.data_ptr(), n, geo.n_video, out.data_ptr(),
         _stream())
    return out


def block_scores(q_means: torch.Tensor, k_means: torch.Tensor, scale: float) -> torch.Tensor:
    q_means, k_means = q_means.contiguous(), k_means.contiguous()
    banks, nb, d = q_means.shape
    out = torch.empty(banks, nb, nb, dtype=torch.float32, device=q_means.device)
    call("recap_block_scores", q_means.data_ptr(), k_means.data_ptr(), banks, nb, d,
         float(scale), out.data_ptr(), _stream())
    return out


def topk_blocks(scores: torch.Tensor, keep: int, force_last: bool) -> torch.Tensor:
    banks, nb, _ = scores.shape
    out = torch.empty(banks, nb, nb, dtype=torch.bool, device=scores.device)
    call("recap_topk_blocks", scores.data_ptr(), banks, nb, int(keep), int(bool(force_last)),
         out.data_ptr(), _stream())
    return out


def kernel_block_mask(partition: torch.Tensor, geo: Geometry) -> torch.Tensor:
    banks = partition.numel() // (geo.nb * geo.nb)
    partition = partition.contiguous()
    out = torch.empty(banks, geo.tb, geo.tb, dtype=torch.bool, device=partition.device)
    call("recap_kernel_block_mask", partition.data_ptr(), banks, geo.n_tokens, geo.n_video,
         out.data_ptr(), _stream())
    return out


def mask_overlap(new: torch.Tensor, old: torch.Tensor) -> tuple[int, int]:
    """(|new & old|, |new|); synchronises the stream to read the counts, as the reference's
    ``float(kept)`` does (recap/operator.py:427)."""
    new, old = new.contiguous(), old.contiguous()
    work = torch.empty(514, dtype=torch.int64, device=new.device)
    call("recap_mask_overlap", new.data_ptr(), old.data_ptr(), new.numel(), work.data_ptr(),
         _stream())
    kept, total = work[:2].tolist()
    return int(kept), int(total)


def pool_select(q: torch.Tensor, k_means: torch.Tensor, rowmap: torch.Tensor, geo: Geometry,
                density: float, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """Stage 1 in one library call: (partition [banks, nb, nb], kernel mask [banks, tb, tb])."""
    b, h, n, d = q.shape
    banks = b * h
    k_means = k_means.contiguous()
    size = int(_lib.load().recap_pool_select_workspace_size(banks, geo.nb, d))
    work = torch.empty(size, dtype=torch.uint8, device=q.device)
    part = torch.empty(banks, geo.nb, geo.nb, dtype=torch.bool, device=q.device)
    kmask = torch.empty(banks, geo.tb, geo.tb, dtype=torch.bool, device=q.device)
    call("recap_pool_select", *_qkv_args(q), rowmap.data_ptr(), n, geo.n_video,
         k_means.data_ptr(), float(scale), float(density), work.data_ptr(), size,
         part.data_ptr(), kmask.data_ptr(), _stream())
    return part, kmask


def select_blocks(q: torch.Tensor, k_means: torch.Tensor, rowmap: torch.Tensor, geo: Geometry,
                  density: float, scale: float) -> torch.Tensor:
    """Partition ``[banks, nb, nb]`` bool (recap/sparse/attention.py:74-94)."""
    q_means = pool_blocks(q, rowmap, geo)
    keep = max(1, round(float(density) * geo.nb))
    keep = min(keep, geo.nb)
    return topk_blocks(block_scores(q_means, k_means, scale), keep, geo.partial)


# -- stage 3 -------------------------------------------------------------------------------


CLOSURE_GROUP = 8


def closure_group(banks: int, nb: int) -> int:
    """Video blocks per closure workgroup: up to CLOSURE_GROUP, fewer when the call has too
    few blocks to give every CU several workgroups (about 1024 in all)."""
    return max(1, min(CLOSURE_GROUP, (banks * nb) // 1024))


@functools.lru_cache(maxsize=256)
def closure_span(banks: int, n_video: int) -> tuple[int, int]:
    """Blocks of a C_vk partial and its runs, for a layer of `banks` heads."""
    group, parts = ctypes.c_int64(), ctypes.c_int64()
    call("recap_closure_span", banks, n_video, ctypes.byref(group), ctypes.byref(parts))
    return group.value, parts.value


def closure_tables(kv: PackedKV, geo: Geometry, basis: "BasisTables", rank: int):
    """The per-call statistics and coarse tables with a frozen basis, in two launches:
    (variance, C_vk in the query type, w, kbar, vbar)."""
    banks, d = kv.k_means.shape[0], kv.dim
    dev = kv.k_means.device
    group, parts = geo.closure_span or closure_span(banks, geo.n_video)
    width = int(_lib.load().recap_coarse_w_width(dtype_code(kv.dtype), d, int(rank)))
    if width < 0:
        raise ValueError(f"closure_tables: invalid dtype/dim/rank ({kv.dtype}, {d}, {rank})")
    for table in (basis.u_hi_t, basis.u_lo_t):
        if table.dtype != kv.dtype or table.numel() != banks * d * d:
            raise ValueError(f"basis table of {table.numel()} {table.dtype} values, expected "
                             f"{banks * d * d} {kv.dtype}")
    padded = -(-geo.nb // COARSE_SLOTS) * COARSE_SLOTS
    partials = int(_lib.load().recap_closure_partials(banks, geo.n_video, group, parts))
    var = torch.empty(banks, geo.nb, d, dtype=torch.float32, device=dev)
    part = torch.empty(partials, d, d, dtype=torch.float32, device=dev)
    cvk_t = torch.empty(banks, d, d, dtype=kv.dtype, device=dev)
    w, kbar, vbar = (torch.empty(banks, padded, c, dtype=kv.dtype, device=dev)
                     for c in (width, d, d))
    call("recap_closure_tables", kv.k_tiles.data_ptr(), kv.vt_tiles.data_ptr(),
         kv.k_means.data_ptr(), kv.v_means.data_ptr(), dtype_code(kv.dtype),
         basis.u_hi_t.data_ptr(), basis.u_lo_t.data_ptr(), banks, d, geo.n_tokens, geo.n_video,
         group, parts, int(rank), var.data_ptr(), part.data_ptr(), cvk_t.data_ptr(),
         w.data_ptr(), kbar.data_ptr(), vbar.data_ptr(), _stream())
    return var, cvk_t, w, kbar, vbar


def closure_stats(kv: PackedKV, geo: Geometry, flags: int, u_hi_t=None, u_lo_t=None,
                  group: int | None = None):
    """(variance, C_vk, scatter) for the requested statistics; absent ones are None."""
    banks, d = kv.k_means.shape[0], kv.dim
    if group is None:
        group = geo.closure_group or closure_group(banks, geo.nb)
    dev = kv.k_means.device
    groups = int(_lib.load().recap_closure_groups(geo.n_video, group))
    var = cvk_part = scat_part = None
    if flags & _lib.CLOSURE_ROT:
        var = torch.empty(banks, geo.nb, d, dtype=torch.float32, device=dev)
    if flags & _lib.CLOSURE_CVK:
        cvk_part = torch.empty(banks, groups, d, d, dtype=torch.float32, device=dev)
    if flags & _lib.CLOSURE_SCATTER:
        scat_part = torch.empty(banks, groups, d, d, dtype=torch.float32, device=dev)
    call("recap_closure_stats", kv.k_tiles.data_ptr(), kv.vt_tiles.data_ptr(),
         kv.k_means.data_ptr(), dtype_code(kv.dtype), _p(u_hi_t), _p(u_lo_t), banks, d,
         geo.n_tokens, geo.n_video, group, flags, _p(var), _p(cvk_part), _p(scat_part), _stream())
    cvk = scatter = None
    if cvk_part is not None:
        cvk = partial_reduce(cvk_part, float(geo.n_video))
    if scat_part is not None:
        scatter = partial_reduce(scat_part, float(geo.n_video))
    return var, cvk, scatter


def partial_reduce(part: torch.Tensor, divisor: float) -> torch.Tensor:
    banks, groups = part.shape[:2]
    elems = part[0, 0].numel()
    out = torch.empty(banks, *part.shape[2:], dtype=torch.float32, device=part.device)
    call("recap_partial_reduce", part.data_ptr(), banks, groups, elems, float(divisor),
         out.data_ptr(), _stream())
    return out


def symmetric_eigen(a: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(eigenvalues ascending ``[..., n]``, eigenvectors as columns ``[..., n, n]``) of the
    symmetrised fp32 ``0.5 (a + a^T)``, n <= 128: the contract of ``torch.linalg.eigh``
    that closure_basis relies on (recap/sparse/closure.py:75-81)."""
    if a.dim() < 2 or a.shape[-1] != a.shape[-2]:
        raise ValueError(f"symmetric_eigen needs square matrices, got {tuple(a.shape)}")
    n = a.shape[-1]
    flat = a.reshape(-1, n, n).to(torch.float32).contiguous()
    values = torch.empty(flat.shape[0], n, dtype=torch.float32, device=a.device)
    vectors = torch.empty_like(flat)
    call("recap_symmetric_eigen", flat.data_ptr(), flat.shape[0], n, values.data_ptr(),
         vectors.data_ptr(), _stream())
    return values.reshape(a.shape[:-1]), vectors.reshape(a.shape)


@dataclass
class BasisTables:
    u_hi_t: torch.Tensor | None = None
    u_lo_t: torch.Tensor | None = None
    u_t: torch.Tensor | None = None
    cvk_t: torch.Tensor | None = None


def basis_tables(basis: torch.Tensor | None, cvk: torch.Tensor | None, dtype: torch.dtype, *,
                 split: bool = False, query: bool = False, cvk_table: bool = False) -> BasisTables:
    basis = None if basis is None else basis.to(torch.float32).contiguous()
    cvk = None if cvk is None else cvk.to(torch.float32).contiguous()
    src = basis if basis is not None else cvk
    banks, d = src.shape[0], src.shape[-1]
    mk = lambda: torch.empty(banks, d, d, dtype=dtype, device=src.device)  # noqa: E731
    out = BasisTables(u_hi_t=mk() if split else None, u_lo_t=mk() if split else None,
                      u_t=mk() if query else None, cvk_t=mk() if cvk_table else None)
    dummy = basis if basis is not None else cvk
    call("recap_basis_tables", dummy.data_ptr(), _p(cvk), dtype_code(dtype), banks, d,
         _p(out.u_hi_t), _p(out.u_lo_t), _p(out.u_t), _p(out.cvk_t), _stream())
    return out


def order_basis(basis: torch.Tensor, var: torch.Tensor, geo: Geometry, dtype: torch.dtype):
    """(basis, variances, tables) with the columns in the order of the pooled within-block
    variance, largest first."""
    banks, nb, d = var.shape
    if basis.shape != (banks, d, d) or nb != geo.nb:
        raise ValueError(f"basis {tuple(basis.shape)} and variances {tuple(var.shape)} do not match")
    basis, var = basis.contiguous(), var.contiguous()
    basis_out, var_out = torch.empty_like(basis), torch.empty_like(var)
    hi, lo, u_t = (torch.empty(banks, d, d, dtype=dtype, device=var.device) for _ in range(3))
    call("recap_order_basis", basis.data_ptr(), var.data_ptr(), dtype_code(dtype), banks, d,
         geo.n_video, basis_out.data_ptr(), var_out.data_ptr(), hi.data_ptr(), lo.data_ptr(),
         u_t.data_ptr(), _stream())
    return basis_out, var_out, BasisTables(u_hi_t=hi, u_lo_t=lo, u_t=u_t)


COARSE_SLOTS = 32  # key blocks per coarse-tail table tile


def coarse_tables(var: torch.Tensor, kv: PackedKV, rank: int):
    """w, kbar, vbar tables [banks, ceil(nb/32)*32, width], one row per key block (see
    recap_coarse_tables; w is [.., 16] in the folded form)."""
    var = var.to(torch.float32).contiguous()
    banks, nb, d = var.shape
    padded = -(-nb // COARSE_SLOTS) * COARSE_SLOTS
    width = int(_lib.load().recap_coarse_w_width(dtype_code(kv.dtype), d, int(rank)))
    if width < 0:
        raise ValueError(f"coarse_tables: invalid dtype/dim/rank ({kv.dtype}, {d}, {rank})")
    mk = lambda c: torch.empty(banks, padded, c, dtype=kv.dtype, device=var.device)  # noqa: E731
    w, kbar, vbar = mk(width), mk(d), mk(d)
    call("recap_coarse_tables", var.data_ptr(), kv.k_means.data_ptr(), kv.v_means.data_ptr(),
         dtype_code(kv.dtype), banks, nb, d, int(rank), w.data_ptr(), kbar.data_ptr(),
         vbar.data_ptr(), _stream())
    return w, kbar, vbar


def coarse_tail(q: torch.Tensor, rowmap: torch.Tensor, partition: torch.Tensor, geo: Geometry,
                tables: dict, scale: float, theta: float, glref: torch.Tensor | None = None):
    """(go [banks, R, d], gl [banks, R], drift partial [banks, R/128] or None).  `tables`
    holds the coarse tables and the closure rank they were built with (key "rank")."""
    for key in ("kbar", "vbar", "w", "u_t", "cvk_t"):
        if tables[key].dtype != q.dtype:
            raise ValueError(f"coarse_tail: table {key} is {tables[key].dtype}, Q is {q.dtype}")
    b, h, n, d = q.shape
    banks = b * h
    partition = partition.contiguous()
    glref = None if glref is None else glref.contiguous()
    go = torch.empty(banks, geo.rows, d, dtype=q.dtype, device=q.device)
    gl = torch.empty(banks, geo.rows, dtype=torch.float32, device=q.device)
    part = None
    if glref is not None:
        part = torch.empty(banks, max(1, geo.rows // BLOCK), dtype=torch.float32, device=q.device)
    call("recap_coarse_tail", *_qkv_args(q), rowmap.data_ptr(), partition.data_ptr(),
         tables["kbar"].data_ptr(), tables["vbar"].data_ptr(), tables["w"].data_ptr(),
         tables["u_t"].data_ptr(), tables["cvk_t"].data_ptr(), n, geo.n_video, float(scale),
         float(theta), int(tables["rank"]), _p(glref), go.data_ptr(), gl.data_ptr(), _p(part),
         _stream())
    return go, gl, part


def drift_center(part: torch.Tensor, geo: Geometry) -> torch.Tensor:
    banks = part.shape[0]
    out = torch.empty(banks, dtype=torch.float32, device=part.device)
    call("recap_drift_center", part.data_ptr(), banks, geo.n_video, out.data_ptr(), _stream())
    return out


# -- stage 2 -------------------------------------------------------------------------------


def block_sparse_attn(q: torch.Tensor, kv: PackedKV, rowmap: torch.Tensor,
                      kernel_mask: torch.Tensor, geo: Geometry, scale: float):
    """Head branch (reordered order): (out [banks, N, d] in the query dtype, lse [banks, N])."""
    _same_type(q, kv)
    b, h, n, d = q.shape
    kernel_mask = kernel_mask.contiguous()
    out = torch.empty(b * h, n, d, dtype=q.dtype, device=q.device)
    lse = torch.empty(b * h, n, dtype=torch.float32, device=q.device)
    split, work = _attn_workspace(q, geo)
    call("recap_block_sparse_attn_ws", *_qkv_args(q), kv.k_tiles.data_ptr(),
         kv.vt_tiles.data_ptr(), rowmap.data_ptr(), kernel_mask.data_ptr(), n, geo.n_video,
         float(scale), out.data_ptr(), lse.data_ptr(), split, 1, work.data_ptr(), work.numel(),
         _stream())
    return out, lse


def attn_split(banks: int, geo: Geometry, density: float = 0.25) -> int:
    """Segments of each long query row for a layer of `banks` heads whose other rows keep about
    `density` of their blocks."""
    return int(_lib.load().recap_attn_split(banks, geo.n_tokens, geo.n_video, float(density)))


@functools.lru_cache(maxsize=256)
def _attn_bytes(*sizes: int) -> int:
    return int(_lib.load().recap_attn_workspace_size(*sizes))


def _attn_workspace(q: torch.Tensor, geo: Geometry) -> tuple[int, torch.Tensor]:
    """(split, workspace) of a masked attention launch."""
    b, h, _, d = q.shape
    split = geo.attn_split or attn_split(b * h, geo)
    size = _attn_bytes(b * h, d, geo.n_tokens, geo.n_video, split)
    if size < 0:
        raise ValueError(f"invalid attention sizes ({geo.n_tokens} tokens, {geo.n_video} video, "
                         f"{d}, split {split})")
    return split, torch.empty(size, dtype=torch.uint8, device=q.device)


def dense_attn(q: torch.Tensor, kv: PackedKV, rowmap: torch.Tensor, scale: float,
               out: torch.Tensor | None = None):
    """Dense attention, native order: (out [B, H, N, d], lse [B, H, N])."""
    _same_type(q, kv)
    b, h, n, d = q.shape
    if out is None:
        out = torch.empty(b, h, n, d, dtype=q.dtype, device=q.device)
    lse = torch.empty(b, h, n, dtype=torch.float32, device=q.device)
    call("recap_dense_attn", *_qkv_args(q), kv.k_tiles.data_ptr(), kv.vt_tiles.data_ptr(),
         rowmap.data_ptr(), n, float(scale), out.data_ptr(), out.stride(0), out.stride(1),
         out.stride(2), lse.data_ptr(), _stream())
    return out, lse


def _work_queue(device, balance: bool):
    """Claim counters for a load-balanced attention launch (zeroed by the call), or None."""
    if not balance:
        return None
    return torch.empty(int(_lib.load().recap_attn_queue_words()), dtype=torch.int32,
                       device=device)


def dense_head_attn(q: torch.Tensor, kv: PackedKV, rowmap: torch.Tensor,
                    kernel_mask: torch.Tensor, scale: float, out: torch.Tensor | None = None,
                    balance: bool = True):
    """A refresh's dense attention and head branch in one pass:
    (out [B, H, N, d] native, lse [B, H, N], head_out [banks, N, d] reordered in the query
    dtype, head_lse [banks, N]).  `balance` lets XCDs that finish early take the others' last query
    blocks (same outputs)."""
    _same_type(q, kv)
    b, h, n, d = q.shape
    kernel_mask = kernel_mask.contiguous()
    if out is None:
        out = torch.empty(b, h, n, d, dtype=q.dtype, device=q.device)
    lse = torch.empty(b, h, n, dtype=torch.float32, device=q.device)
    head_out = torch.empty(b * h, n, d, dtype=q.dtype, device=q.device)
    head_lse = torch.empty(b * h, n, dtype=torch.float32, device=q.device)
    call("recap_dense_head_attn", *_qkv_args(q), kv.k_tiles.data_ptr(), kv.vt_tiles.data_ptr(),
         rowmap.data_ptr(), kernel_mask.data_ptr(), n, float(scale), out.data_ptr(),
         out.stride(0), out.stride(1), out.stride(2), lse.data_ptr(), head_out.data_ptr(),
         head_lse.data_ptr(), _p(_work_queue(q.device, balance)), _stream())
    return out, lse, head_out, head_lse


def sparse_merge_attn(q: torch.Tensor, kv: PackedKV, rowmap: torch.Tensor,
                      kernel_mask: torch.Tensor, geo: Geometry, scale: float, go, gl, det, dl,
                      glref, center, alpha_override: float | None = None,
                      out: torch.Tensor | None = None, balance: bool = True) -> torch.Tensor:
    """Corrected sparse output [B, H, N, d] in native order (one fused kernel); `balance` as
    for dense_head_attn.  ``det`` is fp16 [banks, R, d], or an int8 Microscaled of that shape, read
    in place."""
    _same_type(q, kv)
    b, h, n, d = q.shape
    kernel_mask = kernel_mask.contiguous()
    name, det_args = _refinement("recap_sparse_merge_attn", det, b * h * geo.rows, d, "_ws")
    if any(t is not None and not t.is_contiguous()
           for t in (go, gl, None if name.endswith("_mx") else det, dl, glref, center)):
        raise ValueError("merge inputs must be contiguous")
    if out is None:
        out = torch.empty(b, h, n, d, dtype=q.dtype, device=q.device)
    alpha = -1.0 if alpha_override is None else float(alpha_override)
    split, work = _attn_workspace(q, geo)
    call(name, *_qkv_args(q), kv.k_tiles.data_ptr(),
         kv.vt_tiles.data_ptr(), rowmap.data_ptr(), kernel_mask.data_ptr(), n, geo.n_video,
         float(scale), _p(go), _p(gl), *det_args, _p(dl), _p(glref), _p(center), alpha,
         out.data_ptr(), out.stride(0), out.stride(1), out.stride(2), split, int(balance),
         work.data_ptr(), work.numel(), _stream())
    return out


def _refinement(name: str, det, rows: int, dim: int, plain: str = "") -> tuple[str, tuple]:
    """(entry point, its refinement arguments): fp16 values as they are given, or the codes and
    scales of an int8 Microscaled with `rows` rows of `dim`."""
    if not isinstance(det, Microscaled):
        return name + plain, (_p(det),)
    _refinement_plan(det.format, det.width, rows, dim, *_specs((det.codes, det.scales)))
    return name + "_mx", (det.codes.data_ptr(), det.scales.data_ptr())


@functools.lru_cache(maxsize=256)
def _refinement_plan(format: str, width: int, rows: int, dim: int, codes, scales) -> None:
    """Checks of a microscaled refinement."""
    if format != "int8" or width != dim:
        raise ValueError(f"a refinement is int8 rows of {dim}, got {format} rows of {width}")
    if _check_microscaled("the refinement", "int8", dim, codes, scales) != rows:
        raise ValueError(f"the refinement has {(*codes[0][:-1], width)} values, expected {rows} rows "
                         f"of {dim}")
    _together({"the refinement's codes": codes, "the refinement's scales": scales})


_MASKS, _HALF, _FLOAT = (torch.bool, torch.uint8), (torch.float16,), (torch.float32,)


@functools.lru_cache(maxsize=256)
def _sparse_call_bytes(*sizes: int) -> int:
    return int(_lib.load().recap_sparse_call_workspace_size(*sizes))


def sparse_call(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rowmap: torch.Tensor,
                geo: Geometry, scale: float, theta: float, rank: int, tables: BasisTables,
                partition: torch.Tensor, kernel_mask: torch.Tensor,
                det: "torch.Tensor | Microscaled", dl: torch.Tensor, glref: torch.Tensor,
                alpha_override: float | None = None,
                out: torch.Tensor | None = None, events=None) -> torch.Tensor:
    """A whole corrected sparse call with a frozen basis in one library call and one
    workspace: kv_pack, closure_tables, coarse_tail and sparse_merge_attn with
    their outputs bit for bit, in five launches.  ``det`` as in sparse_merge_attn.  ``events``: five
    timing events recorded before the first stage and after pack, closure (with the tables), coarse
    and attention."""
    if not q.shape == k.shape == v.shape or not q.dtype == k.dtype == v.dtype:
        raise ValueError("Q, K and V must have the same shape and dtype")
    b, h, n, d = q.shape
    if n != geo.n_tokens:
        raise ValueError(f"Q has {n} tokens, the geometry {geo.n_tokens}")
    banks = b * h
    for name in ("u_hi_t", "u_lo_t", "u_t"):
        table = getattr(tables, name)
        if table.dtype != q.dtype:
            raise ValueError(f"coarse_tail: table {name} is {table.dtype}, Q is {q.dtype}")
        if table.numel() != banks * d * d:
            raise ValueError(f"table {name} has {table.numel()} elements, expected {banks * d * d}")
    rows = banks * geo.rows
    entry, det_args = _refinement("recap_sparse_call", det, rows, d)
    half = None if isinstance(det, Microscaled) else det
    for name, t, size, types in (("partition", partition, banks * geo.nb ** 2, _MASKS),
                                 ("kernel_mask", kernel_mask, banks * geo.tb ** 2, _MASKS),
                                 ("det", half, rows * d, _HALF), ("dl", dl, rows, _FLOAT),
                                 ("glref", glref, rows, _FLOAT)):
        if t is not None and (t.numel() != size or t.dtype not in types):
            raise ValueError(f"{name} has {t.numel()} {t.dtype} elements, expected {size} of "
                             f"{types[0]}")
    partition, kernel_mask = partition.contiguous(), kernel_mask.contiguous()
    if not all(t is None or t.is_contiguous() for t in (half, dl, glref)):
        raise ValueError("merge inputs must be contiguous")
    if out is None:
        out = torch.empty(b, h, n, d, dtype=q.dtype, device=q.device)
    code = dtype_code(q.dtype)
    group, parts = geo.closure_span or closure_span(banks, geo.n_video)
    split = geo.attn_split or attn_split(banks, geo)
    size = _sparse_call_bytes(code, banks, d, n, geo.n_video, group, parts, rank, split)
    if size < 0:
        raise ValueError(f"sparse_call: invalid sizes ({n} tokens, {geo.n_video} video, {d}, rank "
                         f"{rank}, group {group}, parts {parts}, split {split})")
    work = torch.empty(size, dtype=torch.uint8, device=q.device)
    handles = None
    if events is not None:
        for event in events:
            event.record()   # creates the event; the call records it again at its stage
        handles = (ctypes.c_void_p * 5)(*(event.cuda_event for event in events))
    call(entry, q.data_ptr(), k.data_ptr(), v.data_ptr(), code, b, h, d,
         *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], rowmap.data_ptr(), n, geo.n_video,
         float(scale), float(theta), rank, group, parts, tables.u_hi_t.data_ptr(),
         tables.u_lo_t.data_ptr(), tables.u_t.data_ptr(), partition.data_ptr(),
         kernel_mask.data_ptr(), *det_args, dl.data_ptr(), glref.data_ptr(),
         -1.0 if alpha_override is None else float(alpha_override), out.data_ptr(),
         *out.stride()[:3], split, handles, work.data_ptr(), size, _stream())
    return out


# -- stage 4 -------------------------------------------------------------------------------


def _check_capture(dense_out, dense_lse, head_out, head_lse, go, gl, det, dl, glref, center):
    """Argument checks shared by both capture entry points: the kernels read the head and
    coarse outputs as 16-bit values of the dense output's type and the refinement as fp16."""
    micro = isinstance(det, Microscaled)
    if not all(t.is_contiguous() for t in (dense_lse, head_out, head_lse, go, gl, dl)) or not (
            micro or det.is_contiguous()):
        raise ValueError("capture inputs must be contiguous")
    if head_out.dtype != dense_out.dtype or go.dtype != dense_out.dtype:
        raise ValueError("capture: head and coarse outputs must have the dense output's dtype")
    if not micro and det.dtype != torch.float16 or dl.dtype != torch.float32:
        raise ValueError("capture: the refinement is fp16 values (or int8 microscaled ones) and fp32 "
                         "log-masses")
    if (glref is None) != (center is None):
        raise ValueError("capture: validation needs both glref and center")


def refresh_capture(dense_out: torch.Tensor, dense_lse: torch.Tensor, head_out: torch.Tensor,
                    head_lse: torch.Tensor, go: torch.Tensor, gl: torch.Tensor,
                    rowmap: torch.Tensor, geo: Geometry, det: "torch.Tensor | Microscaled",
                    dl: torch.Tensor, glref: torch.Tensor | None = None,
                    center: torch.Tensor | None = None):
    """Write the refinement in place; with (glref, center) return the validation pair.  ``det`` is
    fp16 [banks, R, d], or an int8 Microscaled of that shape."""
    b, h, n, d = dense_out.shape
    _check_capture(dense_out, dense_lse, head_out, head_lse, go, gl, det, dl, glref, center)
    name, det_args = _refinement("recap_refresh_capture", det, b * h * geo.rows, d)
    stats = part = None
    if glref is not None:
        npart = int(_lib.load().recap_capture_partials(b * h, d, geo.n_video))
        part = torch.empty(max(1, npart), 2, dtype=torch.float32, device=dense_out.device)
        stats = torch.empty(2, dtype=torch.float32, device=dense_out.device)
    call(name, dense_out.data_ptr(), dtype_code(dense_out.dtype), b, h, d,
         dense_out.stride(0), dense_out.stride(1), dense_out.stride(2), dense_lse.data_ptr(),
         head_out.data_ptr(), head_lse.data_ptr(), go.data_ptr(), gl.data_ptr(),
         rowmap.data_ptr(), n, geo.n_video, *det_args, dl.data_ptr(), _p(glref),
         _p(center), _p(part), _p(stats), _stream())
    return stats


def refresh_capture_noalloc(dense_out: torch.Tensor, dense_lse: torch.Tensor,
                            head_out: torch.Tensor, head_lse: torch.Tensor, go: torch.Tensor,
                            gl: torch.Tensor, rowmap: torch.Tensor, geo: Geometry,
                            det: torch.Tensor, dl: torch.Tensor, stats: torch.Tensor | None,
                            glref: torch.Tensor | None = None,
                            center: torch.Tensor | None = None) -> None:
    """refresh_capture through recap_refresh_capture_noalloc: the library allocates nothing
    (its validation partials live in a static 4 MiB device array); the caller passes the
    validation pair's output ``stats`` ([2] fp32) when validating."""
    b, h, n, d = dense_out.shape
    if isinstance(det, Microscaled):
        raise ValueError("capture: microscaled refinements need refresh_capture")
    _check_capture(dense_out, dense_lse, head_out, head_lse, go, gl, det, dl, glref, center)
    if glref is not None and stats is None:
        raise ValueError("capture: a validating call (glref given) needs the stats output")
    call("recap_refresh_capture_noalloc", dense_out.data_ptr(), dtype_code(dense_out.dtype), b,
         h, d, dense_out.stride(0), dense_out.stride(1), dense_out.stride(2),
         dense_lse.data_ptr(), head_out.data_ptr(), head_lse.data_ptr(), go.data_ptr(),
         gl.data_ptr(), rowmap.data_ptr(), n, geo.n_video, det.data_ptr(), dl.data_ptr(),
         _p(glref), _p(center), _p(stats), _stream())


# -- around the attention call --------------------------------------------------------------

_NORMS = {None: _lib.NORM_NONE, "rms": _lib.NORM_RMS, "layer": _lib.NORM_LAYER}
_QK_NORMS = {**_NORMS, "rms_all": _lib.NORM_RMS_ALL}
_PAIRINGS = {"interleaved": _lib.PAIRS_INTERLEAVED, "halves": _lib.PAIRS_HALVES}
_STREAM_DTYPES = {torch.float16: _lib.RECAP_F16, torch.bfloat16: _lib.RECAP_BF16,
                  torch.float32: _lib.RECAP_F32}


def _choice(table: dict, value, what: str) -> int:
    if value not in table:
        raise ValueError(f"unknown {what} {value!r}; use one of {list(table)}")
    return table[value]


_GRADIENT = "requires a gradient, which this call does not record: run it under torch.no_grad()"
_TANGENT = "carries a forward-mode tangent, which this call does not propagate: unpack it first"


def _specs(tensors) -> tuple:
    """What a call's checks look at of its tensors, hashable: everything but their addresses."""
    grad = torch.is_grad_enabled()
    dual = forward_ad._current_level >= 0
    return tuple([None if t is None else (
        t.shape, t.stride(), t.dtype, t.device,
        _GRADIENT if grad and t.requires_grad else
        _TANGENT if dual and forward_ad.unpack_dual(t).tangent is not None else None)
        for t in tensors])


def _together(specs: dict) -> torch.device:
    """The GPU that all tensors of a call are on.  The kernels have no derivatives, so a call that
    would have to record or propagate one is refused."""
    specs = {name: spec for name, spec in specs.items() if spec is not None}
    for name, spec in specs.items():
        if spec[4]:
            raise ValueError(f"{name} {spec[4]}")
    device = next(iter(specs.values()))[3]
    for name, spec in specs.items():
        if spec[3].type != "cuda":
            raise ValueError(f"{name} must be a GPU tensor")
        if spec[3] != device:
            raise ValueError(f"{name} is on {spec[3]}, the call on {device}")
    return device


def _call_on(device: torch.device, name: str, *args) -> None:
    """Call on the current stream of `device`, which need not be the current device."""
    index = device.index
    if torch._C._cuda_getDevice() == index:
        call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            call(name, *args, torch._C._cuda_getCurrentRawStream(index))


def _span(t: torch.Tensor) -> tuple[int, int]:
    """First and one-past-last byte address of a tensor's elements."""
    last = sum((size - 1) * stride for size, stride in zip(t.shape, t.stride()))
    start = t.data_ptr()
    return start, start + (last + 1) * t.element_size()


def _interleaved(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Two tensors that take turns within rows of one pitch (q and k of a fused projection)
    and share no element."""
    if a.element_size() != b.element_size() or (b.data_ptr() - a.data_ptr()) % a.element_size():
        return False
    steps = [[(st, n) for st, n in zip(t.stride(), t.shape) if n > 1] for t in (a, b)]
    for pitch in {st for st, _ in steps[0]} & {st for st, _ in steps[1]}:
        if any(st > pitch and st % pitch for t in steps for st, _ in t):
            continue
        width_a, width_b = (1 + sum((n - 1) * st for st, n in t if st < pitch) for t in steps)
        shift = (b.data_ptr() - a.data_ptr()) // a.element_size() % pitch
        if width_a <= shift and shift + width_b <= pitch:
            return True
    return False


def _check_output(name: str, out: torch.Tensor, shape, dtype: torch.dtype,
                  inputs: dict[str, torch.Tensor | None], same: str) -> None:
    """A given output: of the right kind, no element of it twice in memory, and over no input's
    memory but that of input `same`, whose exact view it may be."""
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype:
        raise ValueError(f"{name} is {tuple(out.shape)} {out.dtype}, expected {tuple(shape)} "
                         f"{dtype}")
    if out.stride(-1) != 1 and out.shape[-1] > 1:
        raise ValueError(f"{name} must have unit stride along its last dimension")
    extent = 1
    for stride, size in sorted((st, sz) for st, sz in zip(out.stride(), out.shape) if sz > 1):
        if stride < extent:
            raise ValueError(f"{name} has elements that share memory")
        extent += (size - 1) * stride
    if out.numel() == 0:
        return
    lo, hi = _span(out)
    for other, t in inputs.items():
        if t is None or t.numel() == 0:
            continue
        if other == same and t.data_ptr() == lo and t.dtype == dtype and all(
                a == b or n == 1 for a, b, n in zip(t.stride(), out.stride(), out.shape)):
            continue
        start, end = _span(t)
        if start < hi and lo < end and not _interleaved(out, t):
            raise ValueError(f"{name} overlaps the memory of {other}")


def _written(*outs: torch.Tensor | None) -> None:
    """Given outputs count as changed in place, as after torch's own calls: a backward pass that
    saved one before raises instead of using the new values."""
    torch.autograd.graph.increment_version([out for out in outs if out is not None])


def _weights(kind: int, extent: int, dtype: torch.dtype, specs: dict) -> set:
    """Types of the given weights and biases of a norm over `extent` channels."""
    given = {name: v for name, v in specs.items() if v is not None}
    if given and kind == _lib.NORM_NONE:
        raise ValueError(f"{next(iter(given))} needs a norm")
    for name, (shape, _, got, _, _) in given.items():
        if got not in (dtype, torch.float32):
            raise ValueError(f"{name} is {got}; weights and biases are {dtype} or torch.float32")
        if tuple(shape) != (extent,):
            raise ValueError(f"{name} is {tuple(shape)}, expected ({extent},)")
    return {v[2] for v in given.values()}


def _one_type(types: set, dtype: torch.dtype, what: str) -> int:
    if len(types) > 1:
        raise ValueError(f"{what} must have one type, got {sorted(map(str, types))}")
    return _STREAM_DTYPES[next(iter(types), dtype)]


@dataclass(frozen=True)
class _QKPlan:
    """What a qk_rotary call of given shapes, strides and types passes besides addresses."""

    device: torch.device
    copies: bool      # some input is first laid out as the kernel reads it
    empty: bool
    sizes: tuple      # dtype, batch, tokens, dim, heads of q and of k
    lengths: object   # int64 [3], or None without axes
    pairs: object
    codes: tuple      # pairing, norm
    weight_code: int
    strides: tuple    # of q and k, and of outputs made here
    out_strides: tuple


def _aligned_rows(spec) -> bool:
    shape, strides = spec[:2]
    return strides[-1] == 1 and not any(s % 8 for s, n in zip(strides[:3], shape) if n > 1)


def _order(spec) -> tuple:
    """Batch, head and token strides of an output without gaps in its input's order: tokens
    before heads (a projection's) or heads before tokens."""
    (_, h, n, d), (_, by_head, by_token, _) = spec[:2]
    token_major = h > 1 and n > 1 and by_head < by_token
    return (h * n * d, d, h * d) if token_major else (h * n * d, n * d, d)


def _row_strides(shape, strides) -> tuple:
    """Batch, head and token strides; of a dimension of one, whose stride means nothing, d."""
    return tuple(s if n > 1 else shape[3] for s, n in zip(strides[:3], shape))


@functools.lru_cache(maxsize=1024)
def _qk_plan(q, k, axes, offset: int, pairing: str, norm, vectors) -> _QKPlan:
    """Checks of a qk_rotary call, from its tensors' specs."""
    kind = _choice(_QK_NORMS, norm, "norm")
    pairs = _choice(_PAIRINGS, pairing, "pairing")
    for name, spec in (("q", q), ("k", k)):
        if spec is None:
            continue
        if len(spec[0]) != 4:
            raise ValueError(f"{name} must be [batch, heads, tokens, dim], got {tuple(spec[0])}")
        dtype_code(spec[2])
        if spec[0][3] not in (64, 128):
            raise ValueError(f"{name}: head dim {spec[0][3]} unsupported (64 or 128)")
    b, h, n, d = q[0]
    dtype = q[2]
    if k is not None and (k[2] != dtype or k[0][0] != b or k[0][2:] != q[0][2:]):
        raise ValueError(f"K {tuple(k[0])} {k[2]} does not match Q {tuple(q[0])} {dtype}")
    if k is None and not vectors[2] is vectors[3] is None:
        raise ValueError("k_weight and k_bias need a k")
    heads_k = 0 if k is None else k[0][1]
    named = dict(zip(("q_weight", "q_bias", "k_weight", "k_bias"), vectors))
    types = set()
    for heads, prefix in ((h, "q_"), (heads_k, "k_")):
        types |= _weights(kind, heads * d if kind == _lib.NORM_RMS_ALL else d, dtype,
                          {key: v for key, v in named.items() if key.startswith(prefix)})
    weight_code = _one_type(types, dtype, "weights and biases")
    lengths = counts = None
    if axes is not None:
        if len(axes) != 3:
            raise ValueError(f"axes must be three tables (time, height, width), got {len(axes)}")
        for i, (shape, _, got, _, _) in enumerate(axes):
            if len(shape) != 3 or shape[2] != 2 or got != torch.float32 or shape[0] < 1:
                raise ValueError(f"axis {i} must be fp32 [length, channels / 2, 2], got "
                                 f"{tuple(shape)} {got}")
        if sum(t[0][1] for t in axes) != d // 2:
            raise ValueError(f"the axes rotate {[2 * t[0][1] for t in axes]} channels, the heads "
                             f"have {d}")
        video = math.prod(t[0][0] for t in axes)
        if not 0 <= offset <= n - video:
            raise ValueError(f"tokens {offset}..{offset + video - 1} are not all in the sequence "
                             f"of {n}")
        lengths = (ctypes.c_int64 * 3)(*(t[0][0] for t in axes))
        counts = (ctypes.c_int64 * 3)(*(t[0][1] for t in axes))
    tables = axes or ()
    device = _together({"q": q, "k": k, **named, **{f"axis {i}": t for i, t in enumerate(tables)}})
    empty = b * h * n == 0
    if k is not None and empty != (b * heads_k * n == 0):
        raise ValueError("q and k must both have heads")
    copies = not all(_aligned_rows(t) for t in (q, k) if t is not None) or any(
        t[1][0] != 1 and t[0][0] > 1 for t in vectors if t is not None) or any(
        t[1][1:] != (2, 1) or t[1][0] != 2 * t[0][1] for t in tables if t[0][1] > 0)
    return _QKPlan(device, copies, empty, (dtype_code(dtype), b, n, d, h, heads_k), lengths, counts,
                   (pairs, kind), weight_code,
                   tuple((0, 0, 0) if t is None else _row_strides(*t[:2]) for t in (q, k)),
                   tuple((0, 0, 0) if t is None else _order(t) for t in (q, k)))


def qk_rotary(q: torch.Tensor, k: torch.Tensor | None = None, axes=None, *, offset: int = 0,
              pairing: str = "interleaved", norm: str | None = None,
              q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
              q_bias: torch.Tensor | None = None, k_bias: torch.Tensor | None = None,
              eps: float = 1e-6, q_out: torch.Tensor | None = None,
              k_out: torch.Tensor | None = None):
    """Queries and keys for the attention call from their projections: (q, k), k None without
    one.  ``q`` and ``k`` are ``[B, heads, N, d]`` (any strides: views of a projection
    ``[B, N, heads * d]`` or of a fused one are read in place), each with its own heads.

    ``norm`` comes first: ``"rms"`` or ``"layer"`` over a head's channels (weights ``[d]``),
    ``"rms_all"`` over all heads' of a token (weights ``[heads * d]``), or None.  Then the tokens
    ``offset .. offset + T*H*W - 1`` are rotated by their place on the (T, H, W) grid of ``axes``,
    three fp32 tables ``[length, channels / 2, 2]`` of (cos, sin), as recap_amd.rotary_axes makes
    them; the others (text) are not.  ``pairing``: channels ``(2i, 2i + 1)`` (``"interleaved"``) or
    ``(i, i + d / 2)`` (``"halves"``).  ``axes=None`` rotates nothing.

    The outputs have no gaps and keep their input's order in memory (tokens before heads, as a
    projection has them, or heads before tokens).  ``q_out`` and ``k_out`` may be ``q`` and ``k``
    themselves, or views into a longer sequence (a text stream's part of it)."""
    vectors = (q_weight, q_bias, k_weight, k_bias)
    axes = None if axes is None else tuple(axes)
    specs = _specs((q, k, *vectors, *(axes or ())))
    plan = _qk_plan(specs[0], specs[1], None if axes is None else specs[6:], int(offset), pairing,
                    norm, specs[2:6])
    if k is None and k_out is not None:
        raise ValueError("k_out needs a k")
    if q_out is not None or k_out is not None:
        inputs = {"q": q, "k": k, "q_weight": q_weight, "q_bias": q_bias, "k_weight": k_weight,
                  "k_bias": k_bias, **{f"axis {i}": t for i, t in enumerate(axes or ())}}
        _together(dict(zip(("q", "q_out", "k_out"), _specs((q, q_out, k_out)))))
        for name, x, out in (("q", q, q_out), ("k", k, k_out)):
            if out is None:
                continue
            _check_output(f"{name}_out", out, x.shape, x.dtype, inputs, name)
            if not _aligned_rows((out.shape, out.stride())) or out.data_ptr() % 16:
                raise ValueError(f"{name}_out must have 16-byte aligned rows")
        if q_out is not None and k_out is not None:
            _check_output("k_out", k_out, k.shape, k.dtype, {"q_out": q_out}, "")
    strides, out_strides = plan.strides, plan.out_strides
    given = q_out, k_out
    if q_out is not None or k_out is not None:
        out_strides = tuple(made if out is None else _row_strides(out.shape, out.stride())
                            for out, made in zip((q_out, k_out), out_strides))
    if q_out is None:
        q_out = q.new_empty_strided(q.shape, (*out_strides[0], 1))
    if k_out is None and k is not None:
        k_out = k.new_empty_strided(k.shape, (*out_strides[1], 1))
    if plan.empty:
        return q_out, k_out
    if plan.copies or q.data_ptr() % 16 or (k is not None and k.data_ptr() % 16):
        q, k = prepare(q, "q"), None if k is None else prepare(k, "k")
        axes = None if axes is None else tuple(t.contiguous() for t in axes)
        vectors = tuple(None if v is None else v.contiguous() for v in vectors)
        strides = tuple((0, 0, 0) if t is None else _row_strides(t.shape, t.stride())
                        for t in (q, k))
    _call_on(plan.device, "recap_qk_rotary", q.data_ptr(), _p(k), *plan.sizes, *strides[0],
             *strides[1],
             *((None,) * 3 if axes is None else [t.data_ptr() or None for t in axes]), plan.lengths,
             plan.pairs, int(offset), *plan.codes, *map(_p, vectors), plan.weight_code, float(eps),
             q_out.data_ptr(), *out_strides[0], _p(k_out), *out_strides[1])
    if given[0] is not None or given[1] is not None:
        _written(*given)
    return q_out, k_out


def _unit(t: torch.Tensor | None) -> torch.Tensor | None:
    """The tensor with unit stride along its channels, as the kernels read it."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


@dataclass(frozen=True)
class _ResidualPlan:
    """What a residual-stream call of given shapes, strides and types passes besides addresses."""

    device: torch.device
    copies: bool       # some input is first laid out with unit channel stride
    stream: tuple      # type, sizes and strides of x
    branch: tuple      # type and strides of the branch, empty without one
    mods: tuple        # (batch, token) strides of gate, scale and shift
    codes: tuple       # their type, the weights' type, the norms


@functools.lru_cache(maxsize=1024)
def _residual_plan(names, dtype: torch.dtype, x, branch, mods, vectors, norms) -> _ResidualPlan:
    """Checks of a residual-stream call, from its tensors' specs.  ``names``: of the modulation
    and of the weights; ``norms``: (argument, name) of the branch's and the result's norm, each
    with a weight and a bias among ``vectors``."""
    kinds = [_choice(_NORMS, value, what) for what, value in norms]
    shape = tuple(x[0])
    if len(shape) != 3 or shape[2] < 1:
        raise ValueError(f"x must be [batch, tokens, width], got {shape}")
    for got in (x[2], dtype):
        if got not in _STREAM_DTYPES:
            raise ValueError(f"unsupported dtype {got}; use bfloat16, float16 or float32")
    if x[2] not in (dtype, torch.float32):
        raise ValueError(f"a {x[2]} stream goes with a branch and an output of its own type, not "
                         f"{dtype}; a float32 stream goes with any")
    if branch is not None and branch[0] != x[0]:
        raise ValueError(f"branch is {tuple(branch[0])}, the stream {shape}")
    batch, tokens, width = shape
    types, strides = set(), []
    for name, mod in zip(names[0], mods):
        if mod is None:
            strides.append((0, 0))
            continue
        lead, steps = tuple(mod[0][:-1]), mod[1]
        if not 1 <= len(mod[0]) <= 3 or mod[0][-1] != width or not all(
                got in (1, full) for got, full in zip(lead, (batch, tokens))):
            raise ValueError(f"{name} is {tuple(mod[0])}: expected [{width}], [{batch} or 1, {width}] "
                             f"or [{batch} or 1, {tokens} or 1, {width}]")
        if mod[2] not in (dtype, torch.float32):
            raise ValueError(f"{name} is {mod[2]}; gates, scales and shifts are {dtype} or "
                             "torch.float32")
        types.add(mod[2])
        strides.append(tuple([steps[i] if lead[i] > 1 else 0 for i in range(len(lead))]
                             + [0] * (2 - len(lead))))
    mod_code = _one_type(types, dtype, " and ".join(names[0]))
    types = set()
    for i, kind in enumerate(kinds):
        types |= _weights(kind, width, dtype, dict(zip(names[1][2 * i:2 * i + 2],
                                                       vectors[2 * i:2 * i + 2])))
    weight_code = _one_type(types, dtype, "weights and biases")
    device = _together({"x": x, "branch": branch, **dict(zip(names[0], mods)),
                        **dict(zip(names[1], vectors))})
    copies = any(t[1][-1] != 1 and t[0][-1] > 1 for t in (x, branch, *mods, *vectors)
                 if t is not None)
    code = _STREAM_DTYPES[dtype]
    return _ResidualPlan(device, copies, (_STREAM_DTYPES[x[2]], *shape, *x[1][:2]),
                         () if branch is None else (code, *branch[1][:2]), tuple(strides),
                         (mod_code, weight_code, *kinds))


_SCALES, _GATES = ("scale", "shift"), ("gate",)
_AFFINE, _BRANCH_AFFINE = ("weight", "bias"), ("branch_weight", "branch_bias")


def _residual_call(name: str, names, x, dtype, branch, mods, vectors, norms, eps,
                   outs) -> tuple[torch.Tensor, ...]:
    """Checks and launch of the residual-stream calls.  ``outs``: (name, given tensor or None,
    type, the input it may be)."""
    specs = _specs((x, branch, *mods, *vectors))
    last = 2 + len(mods)
    plan = _residual_plan(names, dtype, specs[0], specs[1], specs[2:last], specs[last:], norms)
    made = []
    for out_name, out, out_dtype, same in outs:
        if out is None:
            out = torch.empty_like(x, dtype=out_dtype, memory_format=torch.contiguous_format)
        else:
            inputs = {"x": x, "branch": branch, **dict(zip(names[0], mods)),
                      **dict(zip(names[1], vectors)),
                      **{f"the other output ({o[0]})": m for o, m in zip(outs, made)}}
            _together(dict(zip(("x", out_name), _specs((x, out)))))
            _check_output(out_name, out, x.shape, out_dtype, inputs, same)
        made.append(out)
    if x.numel() == 0:
        return tuple(made)
    if plan.copies:
        return _residual_call(name, names, _unit(x), dtype, _unit(branch), tuple(map(_unit, mods)),
                              tuple(map(_unit, vectors)), norms, eps,
                              [(*o[:1], m, *o[2:]) for o, m in zip(outs, made)])
    args = [x.data_ptr(), *plan.stream]
    if branch is not None:
        args += (branch.data_ptr(), *plan.branch)
    for t, steps in zip(mods, plan.mods):
        args += (_p(t), *steps)
    args += (plan.codes[0], *map(_p, vectors), *plan.codes[1:], float(eps))
    for out in made:
        args += (out.data_ptr(), *out.stride()[:2])
    if branch is None:
        args.insert(-2, _STREAM_DTYPES[dtype])
    _call_on(plan.device, name, *args)
    if any(given is not None for _, given, _, _ in outs):
        _written(*(given for _, given, _, _ in outs))
    return tuple(made)


def norm_modulate(x: torch.Tensor, scale: torch.Tensor | None = None,
                  shift: torch.Tensor | None = None, *, norm: str = "layer",
                  weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                  eps: float = 1e-6, dtype: torch.dtype | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """``norm(x) * (1 + scale) + shift`` of a residual stream ``[B, N, width]``: the norm before a
    block.  ``norm`` is ``"layer"`` or ``"rms"`` over the width, with an optional ``weight`` and
    ``bias``.  ``scale`` and ``shift`` are ``[width]``, ``[B or 1, width]`` or ``[B or 1, N or 1,
    width]``.  ``dtype`` is the output's: x's own, or any for an fp32 stream.  ``out`` may be x
    itself where the types agree."""
    if norm is None:
        raise ValueError("norm must be 'layer' or 'rms'")
    dtype = dtype or x.dtype
    return _residual_call("recap_norm_modulate", (_SCALES, _AFFINE), x, dtype, None, (scale, shift),
                          (weight, bias), (("norm", norm),), eps, [("out", out, dtype, "x")])[0]


def gated_residual(x: torch.Tensor, branch: torch.Tensor, gate: torch.Tensor | None = None, *,
                   branch_norm: str | None = None, branch_weight: torch.Tensor | None = None,
                   branch_bias: torch.Tensor | None = None, eps: float = 1e-6,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """``x + gate * branch_norm(branch)``: a block's output added to the residual stream
    ``[B, N, width]`` (of the branch's type or fp32), after an optional norm of its own.  ``gate``
    has the shapes of norm_modulate's ``scale``; None adds the branch as it is.  ``out`` may be x
    itself."""
    return _residual_call("recap_gated_residual", (_GATES, _BRANCH_AFFINE), x, branch.dtype, branch,
                          (gate,), (branch_weight, branch_bias), (("branch_norm", branch_norm),),
                          eps, [("out", out, x.dtype, "x")])[0]


def gated_residual_norm(x: torch.Tensor, branch: torch.Tensor, gate: torch.Tensor | None = None,
                        scale: torch.Tensor | None = None, shift: torch.Tensor | None = None, *,
                        norm: str = "layer", weight: torch.Tensor | None = None,
                        bias: torch.Tensor | None = None, branch_norm: str | None = None,
                        branch_weight: torch.Tensor | None = None,
                        branch_bias: torch.Tensor | None = None, eps: float = 1e-6,
                        out: torch.Tensor | None = None, norm_out: torch.Tensor | None = None):
    """A block's end and the next one's start in one pass over the residual stream:
    ``r = x + gate * branch_norm(branch)`` and ``norm(r) * (1 + scale) + shift``, as (r, y).  Arguments
    as in gated_residual and norm_modulate; y has the branch's type and is taken from r before
    its rounding.  ``out`` (of r) may be x itself and ``norm_out`` (of y) branch itself."""
    if norm is None:
        raise ValueError("norm must be 'layer' or 'rms'")
    return _residual_call("recap_gated_residual_norm",
                          (_GATES + _SCALES, _BRANCH_AFFINE + _AFFINE), x, branch.dtype, branch,
                          (gate, scale, shift), (branch_weight, branch_bias, weight, bias),
                          (("branch_norm", branch_norm), ("norm", norm)), eps,
                          [("out", out, x.dtype, "x"), ("norm_out", norm_out, branch.dtype, "branch")])


# -- microscaled forms ----------------------------------------------------------------------

MX_BLOCK = 32  # values along a row that share a scale
_MX_FORMATS = {"fp4": _lib.MX_FP4, "int8": _lib.MX_INT8}
_MX_FILL = {"fp4": 256, "int8": MX_BLOCK}
_MX_CODES = {"fp4": torch.uint8, "int8": torch.int8}


@dataclass(frozen=True)
class Microscaled:
    """Rows ``[..., width]`` in 4 or 8 bits, with a power of two for every 32 values along a row.

    ``format`` ``"fp4"``: values 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives times the scale, two
    codes to a byte of ``codes`` (uint8 ``[..., bytes]``); rows are filled up to 256 values.
    ``"int8"``: integers up to 127 times the scale / 64 (int8 ``[..., values]``); rows are filled up
    to 32 values.  ``scales`` (uint8 ``[..., blocks]``) holds each scale's exponent + 127; 255 marks
    a block that held an infinity or NaN and reads as NaN.  Both tensors are contiguous."""

    codes: torch.Tensor
    scales: torch.Tensor
    format: str
    width: int

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.codes.shape[:-1], self.width))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.codes, self.scales))

    @classmethod
    def empty(cls, shape, format: str, device=None) -> "Microscaled":
        """Room for rows of this shape, not yet written."""
        _choice(_MX_FORMATS, format, "format")
        *lead, width = (int(n) for n in shape)
        if width < 1:
            raise ValueError(f"rows of {width} values")
        filled = -(-width // _MX_FILL[format]) * _MX_FILL[format]
        return cls(torch.empty(*lead, filled // 2 if format == "fp4" else filled,
                               dtype=_MX_CODES[format], device=device),
                   torch.empty(*lead, filled // MX_BLOCK, dtype=torch.uint8, device=device),
                   format, width)


def _check_microscaled(name: str, format: str, width: int, codes, scales) -> int:
    """Checks a Microscaled's specs; returns its number of rows."""
    _choice(_MX_FORMATS, format, "format")
    if width < 1:
        raise ValueError(f"{name} has rows of {width} values")
    filled = -(-width // _MX_FILL[format]) * _MX_FILL[format]
    lead = tuple(codes[0][:-1])
    for part, spec, dtype, size in (
            ("codes", codes, _MX_CODES[format], filled // 2 if format == "fp4" else filled),
            ("scales", scales, torch.uint8, filled // MX_BLOCK)):
        if spec[2] != dtype or len(spec[0]) < 1 or tuple(spec[0]) != (*lead, size):
            raise ValueError(f"{name}: {part} of {format} rows of {width} are {dtype} "
                             f"{(*lead, size)}, got {spec[2]} {tuple(spec[0])}")
        step = 1
        for n, stride in zip(reversed(spec[0]), reversed(spec[1])):
            if n > 1 and stride != step and 0 not in lead:
                raise ValueError(f"{name}: {part} must be contiguous")
            step *= n
    return math.prod(lead)


def _even_rows(spec) -> int | None:
    """Stride of the rows of a tensor ``[..., width]``, where one reaches them all."""
    step = size = None
    shape, strides = spec[:2]
    if shape[-1] > 1 and strides[-1] != 1:
        return None
    for n, stride in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if n == 1:
            continue
        if step is None:
            step, size = stride, n
        elif stride != step * size:
            return None
        else:
            size *= n
    return shape[-1] if step is None else step


def _mx_values(name: str, spec) -> None:
    if len(spec[0]) < 1 or spec[0][-1] < 1:
        raise ValueError(f"{name} must be [..., width], got {tuple(spec[0])}")
    if spec[2] not in _STREAM_DTYPES:
        raise ValueError(f"unsupported dtype {spec[2]} of {name}; use bfloat16, float16 or float32")


@functools.lru_cache(maxsize=1024)
def _mx_read_plan(format: str, width: int, codes, scales, dtype: torch.dtype):
    """(device, number of rows, shape) of a microscaled tensor read as dtype."""
    if dtype not in _STREAM_DTYPES:
        raise ValueError(f"unsupported dtype {dtype}; use bfloat16, float16 or float32")
    rows = _check_microscaled("m", format, width, codes, scales)
    return _together({"codes": codes, "scales": scales}), rows, (*codes[0][:-1], width)


@functools.lru_cache(maxsize=1024)
def _mx_rows_plan(name: str, values, format: str, width: int, codes, scales):
    """(device, number of rows, row stride or None) of values [..., width] and their form."""
    _mx_values(name, values)
    lead = tuple(values[0][:-1])
    rows = math.prod(lead)
    if codes is not None:
        _check_microscaled("the microscaled form", format, width, codes, scales)
        if (*lead, width) != (*codes[0][:-1], values[0][-1]):
            raise ValueError(f"{name} is {tuple(values[0])}, the microscaled form "
                             f"{(*codes[0][:-1], width)}")
    device = _together({name: values, "codes": codes, "scales": scales})
    return device, rows, _even_rows(values)


def _aligned(t: torch.Tensor, to: int) -> torch.Tensor:
    return t if t.data_ptr() % to == 0 else t.clone()


def mx_quantise(x: torch.Tensor, format: str = "fp4", *,
                out: Microscaled | None = None) -> Microscaled:
    """Rows ``[..., width]`` of bfloat16, float16 or float32 in their microscaled form.  Each block of
    32 values along a row gets the smallest power of two with which its largest magnitude still
    rounds to a code, and every value its nearest code (ties to the even one).  Rows an even step
    apart (a slice of a wider projection, an expanded row) are read in place, others laid out first.
    ``out`` is written in place: a bank that is kept."""
    _choice(_MX_FORMATS, format, "format")
    specs = _specs((x,) if out is None else (x, out.codes, out.scales))
    if out is not None and out.format != format:
        raise ValueError(f"out is {out.format}, the call's format {format}")
    width = x.shape[-1] if x.ndim else 0
    device, rows, stride = _mx_rows_plan("x", specs[0], format, width if out is None else out.width,
                                         *(specs[1:] or (None, None)))
    given = out
    if out is None:
        out = Microscaled.empty(x.shape, format, device)
    else:
        if out.codes.data_ptr() % 16:
            raise ValueError("out must have 16-byte aligned codes")
        for name, t in (("codes", out.codes), ("scales", out.scales)):
            _apart(f"out's {name}", t, {"x": x})
        _apart("out's codes", out.codes, {"its scales": out.scales})
    if rows == 0:
        return out
    if stride is None:
        x = x.contiguous()
        stride = width
    _call_on(device, "recap_mx_quantise", x.data_ptr(), _STREAM_DTYPES[x.dtype], rows, width, stride,
             _MX_FORMATS[format], out.codes.data_ptr(), out.scales.data_ptr())
    if given is not None:
        _written(given.codes, given.scales)
    return out


def _apart(name: str, out: torch.Tensor, inputs: dict[str, torch.Tensor | None]) -> None:
    if out.numel() == 0:
        return
    lo, hi = _span(out)
    for other, t in inputs.items():
        if t is not None and t.numel():
            start, end = _span(t)
            if start < hi and lo < end and not _interleaved(out, t):
                raise ValueError(f"{name} overlaps the memory of {other}")


def mx_dequantise(m: Microscaled, dtype: torch.dtype = torch.bfloat16, *,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """The values ``[..., width]`` of a microscaled tensor, as ``dtype`` (exact in bfloat16 and
    float32, and in float16 within its range).  ``out``: rows an even step apart."""
    specs = _specs((m.codes, m.scales) if out is None else (m.codes, m.scales, out))
    if out is None:
        device, rows, shape = _mx_read_plan(m.format, m.width, *specs, dtype)
        given, stride = None, m.width
        out = torch.empty(shape, dtype=dtype, device=device)
    else:
        given = out
        device, rows, stride = _mx_rows_plan("out", specs[2], m.format, m.width, *specs[:2])
        _check_output("out", out, m.shape, dtype, {"codes": m.codes, "scales": m.scales}, "")
        if stride is None:
            raise ValueError("out must have rows an even step apart")
    if rows == 0:
        return out
    codes = _aligned(m.codes, 16)
    _call_on(device, "recap_mx_dequantise", codes.data_ptr(), m.scales.data_ptr(),
             _MX_FORMATS[m.format], rows, m.width, out.data_ptr(), _STREAM_DTYPES[out.dtype], stride)
    if given is not None:
        _written(given)
    return out


@dataclass(frozen=True)
class _LinearPlan:
    """What an mx_linear call of given shapes and types passes besides addresses."""

    device: torch.device
    shape: tuple            # of the result
    rows: int
    width: int
    outputs: int
    stride: int | None      # of x's rows; None: x is first laid out
    dtype: torch.dtype      # of the result
    bias_code: int
    workspace: int


@functools.lru_cache(maxsize=1024)
def _linear_plan(x, x_scales, x_form, weight, weight_scales, w_form, bias, dtype) -> _LinearPlan:
    """Checks of an mx_linear call, from its tensors' specs and (format, width) of those in fp4."""
    for name, form in (("x", x_form), ("weight", w_form)):
        if form is not None and form[0] != "fp4":
            raise ValueError(f"{name} is {form[0]}; the product takes fp4 codes")
    outputs = _check_microscaled("weight", *w_form, weight, weight_scales)
    width = w_form[1]
    if len(weight[0]) != 2 or outputs < 1:
        raise ValueError(f"weight must be [outputs, width], got {(*weight[0][:-1], width)}")
    if x_form is not None:
        _check_microscaled("x", *x_form, x, x_scales)
        shape, stride = (*x[0][:-1], x_form[1]), x_form[1]
        dtype = dtype or torch.bfloat16
    else:
        _mx_values("x", x)
        shape, stride = tuple(x[0]), _even_rows(x)
        dtype = dtype or x[2]
    if shape[-1] != width:
        raise ValueError(f"x is {shape}, the weight takes rows of {width}")
    if dtype not in _STREAM_DTYPES:
        raise ValueError(f"unsupported dtype {dtype}; use bfloat16, float16 or float32")
    bias_code = _STREAM_DTYPES[dtype]
    if bias is not None:
        if tuple(bias[0]) != (outputs,):
            raise ValueError(f"bias is {tuple(bias[0])}, expected ({outputs},)")
        if bias[2] not in _STREAM_DTYPES:
            raise ValueError(f"unsupported dtype {bias[2]} of bias")
        bias_code = _STREAM_DTYPES[bias[2]]
    rows = math.prod(shape[:-1])
    device = _together({"x": x, "x's scales": x_scales, "weight": weight,
                        "the weight's scales": weight_scales, "bias": bias})
    size = 0 if rows == 0 or outputs == 0 else int(_lib.load().recap_mx_linear_workspace_size(
        rows, width, outputs, int(x_form is not None)))
    if size < 0:
        raise ValueError(f"mx_linear: {rows} rows of {width} to {outputs} outputs are too many")
    return _LinearPlan(device, (*shape[:-1], outputs), rows, width, outputs, stride, dtype, bias_code,
                       size)


def mx_linear(x: torch.Tensor | Microscaled, weight: Microscaled,
              bias: torch.Tensor | None = None, *, dtype: torch.dtype | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` in 4 bits: ``weight`` is fp4 ``[outputs, width]`` (mx_quantise of a
    projection's weight, once), ``x`` ``[..., width]`` is fp4 too, or a bfloat16, float16 or float32
    tensor that the call brings into fp4.  Several projections of the same rows quantise them once
    and pass the Microscaled.  Products are exact and sums fp32; the result has ``dtype`` (x's own,
    bfloat16 for codes), rounded from fp32 after the bias.  ``out`` may be rows an even step apart (a
    part of a wider tensor)."""
    micro = isinstance(x, Microscaled)
    tensors = (x.codes, x.scales) if micro else (x, None)
    specs = _specs((*tensors, weight.codes, weight.scales, bias))
    plan = _linear_plan(specs[0], specs[1], (x.format, x.width) if micro else None, specs[2],
                        specs[3], (weight.format, weight.width), specs[4], dtype)
    given, stride = out, plan.outputs
    if out is None:
        out = torch.empty(plan.shape, dtype=plan.dtype, device=plan.device)
    else:
        spec = _specs((out,))[0]
        _together({"weight": specs[2], "out": spec})
        _check_output("out", out, plan.shape, plan.dtype,
                      {"x": tensors[0], "x's scales": tensors[1], "weight": weight.codes,
                       "the weight's scales": weight.scales, "bias": bias}, "")
        stride = _even_rows(spec)
        if stride is None:
            raise ValueError("out must have rows an even step apart")
    if plan.rows == 0:
        return out
    codes, scales, x_code, x_stride, work = tensors[0], tensors[1], 0, 0, None
    if micro:
        codes, scales = _aligned(codes, 16), _aligned(scales, 8)
    else:
        x_stride = plan.stride
        if x_stride is None:
            codes, x_stride = x.contiguous(), plan.width
        x_code = _STREAM_DTYPES[x.dtype]
        if plan.workspace:
            work = torch.empty(plan.workspace, dtype=torch.uint8, device=plan.device)
    w, w_scales = _aligned(weight.codes, 16), _aligned(weight.scales, 8)
    bias = _unit(bias)
    _call_on(plan.device, "recap_mx_linear", codes.data_ptr(), x_code, x_stride, _p(scales),
             plan.rows, plan.width, w.data_ptr(), w_scales.data_ptr(), plan.outputs, _p(bias),
             plan.bias_code, out.data_ptr(),
             _STREAM_DTYPES[plan.dtype], stride, _p(work), plan.workspace)
    if given is not None:
        _written(given)
    return out


def bank_copy_async(dst: torch.Tensor, src: torch.Tensor, stream=None) -> None:
    """Asynchronous device <-> pinned-host copy of a whole bank tensor on ``stream``."""
    if dst.numel() * dst.element_size() != src.numel() * src.element_size():
        raise ValueError("bank copy size mismatch")
    if not (dst.is_contiguous() and src.is_contiguous()):
        raise ValueError("bank copies need contiguous tensors")
    handle = (stream or torch.cuda.current_stream()).cuda_stream
    call("recap_bank_copy_async", dst.data_ptr(), src.data_ptr(),
         dst.numel() * dst.element_size(), handle)


def hilbert_permutation_native(grid) -> "torch.Tensor":
    frames, height, width = (int(x) for x in grid)
    out = torch.empty(frames * height * width, dtype=torch.int64)
    call("recap_hilbert_permutation", frames, height, width, out.data_ptr())
    return out


def scale_for(dim: int) -> float:
    return 1.0 / math.sqrt(dim)
