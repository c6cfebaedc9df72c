"""Drop-in for the reference's pybind11 module ``CudaGaussianVoxelizer._C`` (src/bindings.cpp:7-64).

Same function names, keyword arguments, tuple layouts and error behaviour (``RuntimeError``)
as the reference; the work is done by libg2v_hip.so through its C ABI (include/g2v.h) on the
caller's current HIP stream.  Outputs and workspaces come from PyTorch's caching allocator.
"""
from __future__ import annotations

import array
import ctypes
import functools
import math
import operator

import torch

from . import _lib

__all__ = ["gaussian_voxelizer_forward", "gaussian_voxelizer_backward", "gaussian_voxelizer_forward_batched",
           "CudaFeatsCosinelossForward", "CudaFeatsCosinelossBackward", "build_t2g", "grid_dims",
           "covariance_from_scale_rotation", "covariance_from_scale_rotation_backward",
           "qk_norm_rotary_forward", "qk_norm_rotary_backward", "attention_forward", "attention_backward"]


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _host_values(t, n, name):
    """Host floats of voxel_size / voxel_range.  Device tensors are read once per version."""
    if isinstance(t, torch.Tensor):
        if t.numel() != n:
            raise RuntimeError(f"{name} must have {n} elements, got {t.numel()}")
        if t.device.type == "cpu":
            return [float(v) for v in t.detach().reshape(-1).to(torch.float32).tolist()]
        cached = t.__dict__.get("_g2v_host")
        if cached is not None and cached[0] == t._version:
            return cached[1]
        vals = [float(v) for v in t.detach().reshape(-1).to(torch.float32).cpu().tolist()]
        t.__dict__["_g2v_host"] = (t._version, vals)
        return vals
    vals = [float(v) for v in t]
    if len(vals) != n:
        raise RuntimeError(f"{name} must have {n} elements, got {len(vals)}")
    return vals


def grid_dims(voxel_size, voxel_range):
    """((X, Y, Z), (Tx, Ty, Tz)) as the forward computes them (reference .cu:1511-1519)."""
    lib = _lib.load()
    vs = _lib.floats(_host_values(voxel_size, 3, "voxel_size"))
    vr = _lib.floats(_host_values(voxel_range, 6, "voxel_range"))
    dims = (ctypes.c_int * 3)()
    tiles = (ctypes.c_int * 3)()
    _lib.check(lib.g2v_grid_dims(vs, vr, dims, tiles), "g2v_grid_dims")
    return tuple(dims), tuple(tiles)


_GRIDS = {}


def _grid_of(voxel_size, voxel_range):
    """(vs, vr, dims, tiles) of a grid: the ctypes float arrays the C ABI takes and the grid and tile
    dimensions, kept per distinct (voxel_size, voxel_range) values."""
    vs_h = _host_values(voxel_size, 3, "voxel_size")
    vr_h = _host_values(voxel_range, 6, "voxel_range")
    key = tuple(vs_h) + tuple(vr_h)
    g = _GRIDS.get(key)
    if g is None:
        dims, tiles = grid_dims(vs_h, vr_h)
        g = (_lib.floats(vs_h), _lib.floats(vr_h), dims, tiles)
        if len(_GRIDS) < 64:
            _GRIDS[key] = g
    return g


def _f32_input(t, name, shape=None):
    if isinstance(t, torch.Tensor) and t.dtype == torch.float32 \
            and t.is_cuda and t.is_contiguous() and (shape is None or t.shape == shape):
        return t.detach()   # already what the kernels read
    return _f32_input_slow(t, name, shape)


def _f32_input_slow(t, name, shape=None):
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor")
    if t.device.type != "cuda":
        raise RuntimeError(f"{name} must be a GPU tensor, got {t.device}")
    if t.dtype != torch.float32:
        raise RuntimeError(f"expected scalar type Float for {name} but found {t.dtype}")
    if shape is not None:
        t = t.reshape(shape)
    return t.detach().contiguous()


_FEAT_DTYPES = {torch.float32: _lib.G2V_DTYPE_F32, torch.bfloat16: _lib.G2V_DTYPE_BF16}


def _feat_input(t, name):
    """Features: float32 or bfloat16 on the GPU (grid_feats and the feature gradient take the
    same type)."""
    if isinstance(t, torch.Tensor) and t.dtype in _FEAT_DTYPES and t.is_cuda and t.is_contiguous():
        return t.detach()
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor")
    if t.device.type != "cuda":
        raise RuntimeError(f"{name} must be a GPU tensor, got {t.device}")
    if t.dtype not in _FEAT_DTYPES:
        raise RuntimeError(f"expected scalar type Float or BFloat16 for {name} but found {t.dtype}")
    return t.detach().contiguous()


def _check_saved(t, name, dtype, device):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or not t.is_contiguous() or t.device != device:
        raise RuntimeError(f"{name} must be a contiguous {dtype} tensor on {device}")


def _stream(device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


_EVENTS = {}
_READY = {}


def _timing_events(device):
    """A (start, stop) pair of timing events per device and thread, reused by every call (each call
    records and synchronises both before it returns)."""
    import threading
    key = (device.index, threading.get_ident())
    ev = _EVENTS.get(key)
    if ev is None:
        ev = (torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True))
        _EVENTS[key] = ev
    return ev


def _ready_event(device):
    """An event per device and thread that marks where a host wait ends (no timing)."""
    import threading
    key = (device.index, threading.get_ident())
    ev = _READY.get(key)
    if ev is None:
        ev = torch.cuda.Event()
        _READY[key] = ev
    return ev


class _OnDevice:
    """torch.cuda.device(dev) only when dev is not already the current device."""

    def __init__(self, dev):
        self.ctx = None if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *exc):
        if self.ctx is not None:
            self.ctx.__exit__(*exc)
        return False


def gaussian_voxelizer_forward(means3D, opacity, covariances, voxel_size, voxel_range, features=None):
    """Gaussian voxelization forward pass.

    Args:
        means3D (N,3), opacity (N,) (or (N,1)), covariances (N,9) row-major 3x3 (or (N,3,3)),
        voxel_size (3,), voxel_range (6,) [x_min, y_min, z_min, x_max, y_max, z_max],
        features (N,C) or None.  All float32 on the GPU.
    Returns the reference's 9-tuple (src/cuda_gaussian_voxelizer.cu:1913):
        density (X,Y,Z), cov_inv (N,9), valid_voxel_lb (N,3) int32, valid_voxel_ub (N,3) int32,
        num_voxels_per_gaussian (N,) int32, grid_feats (X,Y,Z,C) (C = 0 without features),
        g2t_offsets (N+1,) int32, g2t_tile_ids (M,) int32, forward time in seconds.
    """
    return _forward(means3D, opacity, covariances, voxel_size, voxel_range, features, keep_t2g=False)[0]


def _forward(means3D, opacity, covariances, voxel_size, voxel_range, features, keep_t2g):
    """The forward; with keep_t2g it also returns, beside the 9-tuple, what the backward would
    otherwise recompute: the Tile->Gaussian CSR (sorted tiles, sorted Gaussians, tile offsets) and
    the backward plan (region pair offsets and their count, counted on the plan's one sync)."""
    lib = _lib.load()
    means = _f32_input(means3D, "means3D")
    if means.dim() != 2 or means.shape[1] != 3:
        raise RuntimeError(f"means3D must be (N, 3), got {tuple(means.shape)}")
    n = means.shape[0]
    dev = means.device
    op = _f32_input(opacity, "opacity", (n,))
    cov = _f32_input(covariances, "covariances", (n, 9))
    feats = None
    C = 0
    if features is not None:
        feats = _feat_input(features, "features")
        if feats.dim() != 2 or feats.shape[0] != n:
            raise RuntimeError(f"features must be (N, C) with N = {n}, got {tuple(feats.shape)}")
        C = feats.shape[1]
        if C == 0:
            feats = None
    vs, vr, (X, Y, Z), (Tx, Ty, Tz) = _grid_of(voxel_size, voxel_range)

    with _OnDevice(dev):
        cur = torch.cuda.current_stream(dev)
        stream = ctypes.c_void_p(cur.cuda_stream)
        i32 = dict(dtype=torch.int32, device=dev)
        f32 = dict(dtype=torch.float32, device=dev)
        cov_inv = torch.empty(n, 9, **f32)
        lb = torch.empty(n, 3, **i32)
        ub = torch.empty(n, 3, **i32)
        nvox = torch.empty(n, **i32)
        g2t_offsets = torch.empty(n + 1, **i32)
        # the plan's workspace and, with keep_t2g, the backward plan's (the (region, Gaussian) pair
        # count is done here too, on the same wait; the backward reads that workspace later), in
        # one allocation
        pws = lib.g2v_forward_plan_workspace(n)
        pws_al = (pws + 255) & ~255
        # (without features the backward needs neither the CSR nor a plan: it walks the boxes)
        keep_csr = keep_t2g and feats is not None
        bws = max(1, lib.g2v_backward_plan_workspace(n)) if keep_csr else 0
        wsb = torch.empty(pws_al + bws, dtype=torch.uint8, device=dev)
        ws = wsb[:pws]
        bplan = wsb[pws_al:] if keep_csr else None
        counts = _pinned_counts(dev, 2)
        start, stop = _timing_events(dev)
        start.record(cur)
        _lib.check(lib.g2v_forward_plan_async(n, _ptr(means), _ptr(cov), vs, vr, _ptr(cov_inv), _ptr(lb),
                                              _ptr(ub), _ptr(nvox), _ptr(g2t_offsets), _ptr(ws), ws.numel(),
                                              _ptr(bplan), 0 if bplan is None else bplan.numel(), _ptr(counts),
                                              stream),
                   "gaussian_voxelizer_forward (plan)")
        ready = _ready_event(dev)
        ready.record(cur)
        # queued behind the plan, so that they run while this thread waits for the pair counts:
        # the features packed for the splat; then the outputs whose size does not depend on the
        # counts are allocated
        fdtype = torch.float32 if feats is None else feats.dtype
        fdt = _FEAT_DTYPES[fdtype]
        packed = None
        if feats is not None:
            packed = torch.empty(lib.g2v_forward_packed_bytes(n, C), dtype=torch.uint8, device=dev)
            _lib.check(lib.g2v_forward_pack_features(n, C, _ptr(feats), fdt, _ptr(packed), packed.numel(), stream),
                       "gaussian_voxelizer_forward (features)")
        density = torch.empty(X, Y, Z, **f32)
        grid_feats = torch.empty(X, Y, Z, C, dtype=fdtype, device=dev)
        t2g_toff = torch.empty(Tx * Ty * Tz + 1, **i32) if keep_csr else None
        ready.synchronize()
        M, MR = (int(v) for v in counts.tolist())
        for cnt, what in ((M, "Gaussian-tile"), (MR, "region-Gaussian")):
            if cnt > 2147483647:
                raise RuntimeError(f"gaussian_voxelizer_forward (plan): {cnt} {what} pairs exceed the int32 CSR "
                                   "(limit 2^31-1)")
        g2t_tile_ids = torch.empty(M, **i32)
        ws2 = torch.empty(lib.g2v_forward_splat_workspace(n, C, M, vs, vr), dtype=torch.uint8, device=dev)
        t2g = None
        csr = (None, None, None)
        if keep_t2g:
            if keep_csr:
                csr = (torch.empty(M, **i32), torch.empty(M, **i32), t2g_toff)
            t2g = dict(csr=csr, plan=bplan, num_region_pairs=MR, vs=vs, vr=vr, dims=(X, Y, Z))
        _lib.check(lib.g2v_forward_splat(n, C, _ptr(means), _ptr(op), _ptr(feats), fdt, _ptr(packed),
                                         0 if packed is None else packed.numel(), vs, vr,
                                         _ptr(cov_inv), _ptr(lb), _ptr(ub), _ptr(g2t_offsets), M,
                                         _ptr(g2t_tile_ids), _ptr(density), _ptr(grid_feats),
                                         _ptr(csr[0]), _ptr(csr[1]), _ptr(csr[2]),
                                         _ptr(ws2), ws2.numel(), stream),
                   "gaussian_voxelizer_forward (splat)")
        stop.record(cur)
        if keep_t2g:
            # the backward's outputs and workspace, allocated while the forward kernels run
            t2g["grads"] = (torch.empty(n, 3, **f32), torch.empty(n, 9, **f32), torch.empty(n, **f32),
                            torch.empty(n, C, dtype=fdtype, device=dev))
            t2g["ws"] = torch.empty(max(1, lib.g2v_backward_workspace(n, C, M, t2g["num_region_pairs"], vs, vr)),
                                    dtype=torch.uint8, device=dev) if C > 0 else None
            # the backward's gradient-independent kernels, queued behind the forward (after its
            # stop event): they run while this thread waits and hands over to the backward
            if C > 0:
                _lib.check(lib.g2v_backward_prepare(n, C, vs, vr, _ptr(lb), _ptr(ub), _ptr(feats), fdt, M,
                                                    t2g["num_region_pairs"], _ptr(csr[0]), _ptr(csr[1]),
                                                    _ptr(bplan), _ptr(t2g["ws"]), t2g["ws"].numel(), stream),
                           "gaussian_voxelizer_forward (backward preparation)")
                t2g["prepared"] = True
        stop.synchronize()
        fwd_sec = start.elapsed_time(stop) / 1000.0
    return (density, cov_inv, lb, ub, nvox, grid_feats, g2t_offsets, g2t_tile_ids, fwd_sec), t2g


def gaussian_voxelizer_backward(grad_output, grad_feats_output, means3D, opacity, cov_inv, voxel_size,
                                voxel_range, valid_voxel_lb, valid_voxel_ub, num_voxels_per_gaussian,
                                g2t_offsets, g2t_tile_ids, density, grid_feats, features=None):
    """Gaussian voxelization backward pass (reference src/cuda_gaussian_voxelizer.cu:1920-2057).

    Returns the reference's 5-tuple: grad_means (N,3), grad_cov (N,9), grad_opacity (N,),
    grad_feats (N,C) (N,0 without features), backward time in seconds.
    """
    return _backward(grad_output, grad_feats_output, means3D, opacity, cov_inv, voxel_size, voxel_range,
                     valid_voxel_lb, valid_voxel_ub, num_voxels_per_gaussian, g2t_offsets, g2t_tile_ids,
                     density, grid_feats, features, t2g=None)


def gaussian_voxelizer_backward_cosine(grad_output, grad_loss, pseudo_dino_gt, coef, num_valid_voxel, means3D,
                                       opacity, cov_inv, voxel_size, voxel_range, valid_voxel_lb, valid_voxel_ub,
                                       num_voxels_per_gaussian, g2t_offsets, g2t_tile_ids, density, grid_feats,
                                       features):
    """gaussian_voxelizer_backward with the feature cosine loss's gradient as the upstream gradient
    of grid_feats, fused (g2v_backward_cosine): the (X,Y,Z,C) gradient that the reference's
    CudaFeatsCosinelossBackward writes and its voxelizer backward reads (src/cuda_feats_loss.cu:
    311-366, src/cuda_gaussian_voxelizer.cu:1920-2057) is formed per voxel inside the kernels.
    grad_loss: the upstream gradient of the loss (one-element GPU tensor); coef and num_valid_voxel
    as _cosine_forward(..., want_coef=True) returned them for this grid_feats and pseudo_dino_gt
    (float32, C % 4 == 0).  Returns gaussian_voxelizer_backward's 5-tuple."""
    gl = grad_loss.detach().to(device=means3D.device, dtype=torch.float32).reshape(1).contiguous()
    return _backward(grad_output, None, means3D, opacity, cov_inv, voxel_size, voxel_range, valid_voxel_lb,
                     valid_voxel_ub, num_voxels_per_gaussian, g2t_offsets, g2t_tile_ids, density, grid_feats,
                     features, t2g=None, cosine=(gl, pseudo_dino_gt, coef, num_valid_voxel))


def _backward(grad_output, grad_feats_output, means3D, opacity, cov_inv, voxel_size, voxel_range,
              valid_voxel_lb, valid_voxel_ub, num_voxels_per_gaussian, g2t_offsets, g2t_tile_ids,
              density, grid_feats, features, t2g, timed=True, cosine=None):
    """The backward; t2g is what _forward(keep_t2g=True) returned beside the 9-tuple, or None.
    With t2g the saved tensors are the forward's own outputs (already checked there), and the
    grid, plan, outputs and workspace come from the forward: only the upstream gradients are
    checked here.  cosine = (grad_loss, pseudo_dino_gt, coef, num_valid_voxel): the upstream
    gradient of grid_feats is the cosine loss's, formed inside the kernels (grad_feats_output is
    ignored)."""
    lib = _lib.load()
    if not isinstance(means3D, torch.Tensor) or means3D.device.type != "cuda":
        raise RuntimeError("means3D must be a GPU tensor")
    dev = means3D.device
    f32, i32 = torch.float32, torch.int32
    trusted = t2g is not None and "grads" in t2g
    if trusted:
        vs, vr = t2g["vs"], t2g["vr"]
        X, Y, Z = t2g["dims"]
        _check_saved(grad_output, "grad_output", f32, dev)
    else:
        for t, name in ((grad_output, "grad_output"), (means3D, "means3D"), (opacity, "opacity"),
                        (cov_inv, "cov_inv"), (density, "density")):
            _check_saved(t, name, f32, dev)
        _check_saved(grid_feats, "grid_feats", grid_feats.dtype if grid_feats.dtype in _FEAT_DTYPES else f32, dev)
        for t, name in ((valid_voxel_lb, "valid_voxel_lb"), (valid_voxel_ub, "valid_voxel_ub"),
                        (num_voxels_per_gaussian, "num_voxels_per_gaussian"), (g2t_offsets, "g2t_offsets"),
                        (g2t_tile_ids, "g2t_tile_ids")):
            _check_saved(t, name, i32, dev)
        vs_h = _host_values(voxel_size, 3, "voxel_size")
        vr_h = _host_values(voxel_range, 6, "voxel_range")
        vs, vr = _lib.floats(vs_h), _lib.floats(vr_h)
        (X, Y, Z), _ = grid_dims(vs_h, vr_h)
    n = means3D.shape[0]
    if g2t_offsets.numel() != n + 1:
        raise RuntimeError(f"g2t_offsets must have N+1 = {n + 1} elements, got {g2t_offsets.numel()}")
    if tuple(grad_output.shape) != (X, Y, Z):
        raise RuntimeError(f"grad_output must be {(X, Y, Z)}, got {tuple(grad_output.shape)}")
    C = 0
    feats = gF = None
    fdtype = f32
    if features is not None:
        if not trusted:
            _check_saved(features, "features", features.dtype if features.dtype in _FEAT_DTYPES else f32, dev)
        C = features.shape[1]
        fdtype = features.dtype
        if C > 0:
            feats = features
            if grid_feats.dtype != fdtype:
                raise RuntimeError(f"grid_feats ({grid_feats.dtype}) and features ({fdtype}) differ in type")
            if cosine is not None:
                grad_feats_output = cosine[1]   # checked as the stand-in upstream tensor
                coef, gl = cosine[2], cosine[0]
                _check_saved(coef, "coef", f32, dev)
                _check_saved(gl, "grad_loss", f32, dev)
                if tuple(coef.shape) != (X * Y * Z, 2) or gl.numel() != 1:
                    raise RuntimeError(f"coef must be ({X * Y * Z}, 2) and grad_loss one element")
                if fdtype != f32 or C % 4 != 0:
                    raise RuntimeError("the fused cosine gradient takes float32 features with C % 4 == 0")
            else:
                # the upstream feature gradient is taken in the features' type (a float32 gradient of
                # bfloat16 features is rounded to bfloat16, a bfloat16 one of float32 features widened)
                if isinstance(grad_feats_output, torch.Tensor) and grad_feats_output.dtype != fdtype \
                        and grad_feats_output.dtype in _FEAT_DTYPES:
                    grad_feats_output = grad_feats_output.to(fdtype).contiguous()
            _check_saved(grad_feats_output, "pseudo_dino_gt" if cosine is not None else "grad_feats_output",
                         fdtype, dev)
            if tuple(grad_feats_output.shape) != (X, Y, Z, C) or tuple(grid_feats.shape) != (X, Y, Z, C):
                raise RuntimeError("grad_feats_output and grid_feats must be (X, Y, Z, C)")
            gF = grad_feats_output
    fdt = _FEAT_DTYPES[fdtype]
    M = g2t_tile_ids.numel()

    with _OnDevice(dev):
        cur = torch.cuda.current_stream(dev)
        stream = ctypes.c_void_p(cur.cuda_stream)
        if trusted:   # allocated by the forward
            grad_means, grad_cov, grad_opacity, grad_feats = t2g["grads"]
        else:
            grad_means = torch.empty(n, 3, dtype=f32, device=dev)
            grad_cov = torch.empty(n, 9, dtype=f32, device=dev)
            grad_opacity = torch.empty(n, dtype=f32, device=dev)
            grad_feats = torch.empty(n, C, dtype=fdtype, device=dev)
        if timed:
            start, stop = _timing_events(dev)
            start.record(cur)
        if C == 0:   # the density-only backward walks the boxes: no plan, no workspace
            plan_ws, MR = None, 0
        elif t2g is not None:   # planned by the forward
            plan_ws, MR = t2g["plan"], t2g["num_region_pairs"]
        else:
            plan_ws = torch.empty(max(1, lib.g2v_backward_plan_workspace(n)), dtype=torch.uint8, device=dev)
            MR = ctypes.c_longlong(0)
            _lib.check(lib.g2v_backward_plan(n, C, vs, vr, _ptr(valid_voxel_lb), _ptr(valid_voxel_ub),
                                             _ptr(plan_ws), plan_ws.numel(), ctypes.byref(MR), stream),
                       "gaussian_voxelizer_backward (plan)")
            MR = int(MR.value)
        if C == 0:
            ws = None
        elif trusted:
            ws = t2g["ws"]
        else:
            ws = torch.empty(max(1, lib.g2v_backward_workspace(n, C, M, MR, vs, vr)), dtype=torch.uint8, device=dev)
        csr = t2g["csr"] if t2g else (None, None, None)
        # the forward queued the gradient-independent part into this workspace
        prepared = bool(trusted and C > 0 and t2g.get("prepared"))
        if cosine is not None and C > 0:
            grad_loss, _, coef, num_valid = cosine
            _lib.check(lib.g2v_backward_cosine(n, C, _ptr(grad_output), _ptr(grad_loss), _ptr(gF), _ptr(coef),
                                               int(num_valid), _ptr(means3D), _ptr(opacity), _ptr(cov_inv), vs, vr,
                                               _ptr(valid_voxel_lb), _ptr(valid_voxel_ub),
                                               _ptr(num_voxels_per_gaussian), _ptr(g2t_offsets),
                                               _ptr(g2t_tile_ids), M, MR, _ptr(density), _ptr(grid_feats),
                                               _ptr(feats), fdt, _ptr(grad_means), _ptr(grad_cov),
                                               _ptr(grad_opacity), _ptr(grad_feats), _ptr(csr[0]), _ptr(csr[1]),
                                               _ptr(csr[2]), _ptr(plan_ws), _ptr(ws), ws.numel(), int(prepared),
                                               stream),
                       "gaussian_voxelizer_backward_cosine")
        else:
            entry = lib.g2v_backward_prepared if prepared else lib.g2v_backward
            _lib.check(entry(n, C, _ptr(grad_output), _ptr(gF), _ptr(means3D), _ptr(opacity),
                             _ptr(cov_inv), vs, vr, _ptr(valid_voxel_lb), _ptr(valid_voxel_ub),
                             _ptr(num_voxels_per_gaussian), _ptr(g2t_offsets), _ptr(g2t_tile_ids),
                             M, MR, _ptr(density), _ptr(grid_feats), _ptr(feats), fdt,
                             _ptr(grad_means), _ptr(grad_cov), _ptr(grad_opacity),
                             _ptr(grad_feats), _ptr(csr[0]), _ptr(csr[1]), _ptr(csr[2]),
                             _ptr(plan_ws), _ptr(ws), 0 if ws is None else ws.numel(), stream),
                       "gaussian_voxelizer_backward")
        bwd_sec = 0.0
        if timed:
            stop.record(cur)
            stop.synchronize()
            bwd_sec = start.elapsed_time(stop) / 1000.0
    return (grad_means, grad_cov, grad_opacity, grad_feats, bwd_sec)


_COUNTS = {}


def _pinned_counts(dev, k):
    """A reusable pinned (k,) int64 host buffer per device and thread (count read-back)."""
    import threading
    key = (dev.index, threading.get_ident())
    buf = _COUNTS.get(key)
    if buf is None or buf.numel() < k:
        buf = torch.empty(max(k, 16), dtype=torch.int64, pin_memory=True)
        _COUNTS[key] = buf
    return buf[:k]


def gaussian_voxelizer_forward_batched(means3D, opacity, covariances, voxel_size, voxel_range, features=None):
    """Forward of B scenes on one grid in one call: means3D (B,N,3), opacity (B,N) or (B,N,1),
    covariances (B,N,9) or (B,N,3,3), features (B,N,C) or None.

    The B scenes run as one problem of B N Gaussians (one launch per kernel for the whole batch,
    one host wait for its pair counts).  Returns a list of B 9-tuples laid out as
    gaussian_voxelizer_forward's, each equal to that of the scene alone; the density and
    grid_feats of scene b are the views [b] of one (B,X,Y,Z) and one (B,X,Y,Z,C) tensor, and the
    time in every tuple is that of the whole batch.
    """
    return _forward_batched(means3D, opacity, covariances, voxel_size, voxel_range, features, keep_t2g=False)[0]


def _forward_batched(means3D, opacity, covariances, voxel_size, voxel_range, features, keep_t2g):
    """Batched forward.  Returns ([9-tuple per scene], density (B,X,Y,Z), grid_feats (B,X,Y,Z,C),
    batch) where batch holds what _backward_batched needs (the batch plan, the batch's
    Tile->Gaussian CSR, the prepared backward workspace) with keep_t2g, else None."""
    lib = _lib.load()
    means = _f32_input(means3D, "means3D")
    if means.dim() != 3 or means.shape[2] != 3:
        raise RuntimeError(f"batched means3D must be (B, N, 3), got {tuple(means.shape)}")
    B, n = means.shape[0], means.shape[1]
    dev = means.device
    op = _f32_input(opacity, "opacity", (B, n))
    cov = _f32_input(covariances, "covariances", (B, n, 9))
    feats = None
    C = 0
    if features is not None:
        feats = _feat_input(features, "features")
        if feats.dim() != 3 or tuple(feats.shape[:2]) != (B, n):
            raise RuntimeError(f"features must be (B, N, C) with B, N = {B}, {n}, got {tuple(feats.shape)}")
        C = feats.shape[2]
        if C == 0:
            feats = None
    vs_h = _host_values(voxel_size, 3, "voxel_size")
    vr_h = _host_values(voxel_range, 6, "voxel_range")
    vs, vr = _lib.floats(vs_h), _lib.floats(vr_h)
    (X, Y, Z), (Tx, Ty, Tz) = grid_dims(vs_h, vr_h)
    T = Tx * Ty * Tz
    if B == 0:
        f32 = dict(dtype=torch.float32, device=dev)
        return [], torch.empty(0, X, Y, Z, **f32), torch.empty(0, X, Y, Z, C, dtype=torch.float32 if feats is None
                                                                 else feats.dtype, device=dev), None

    with _OnDevice(dev):
        cur = torch.cuda.current_stream(dev)
        stream = ctypes.c_void_p(cur.cuda_stream)
        i32 = dict(dtype=torch.int32, device=dev)
        f32 = dict(dtype=torch.float32, device=dev)
        cov_inv = torch.empty(B, n, 9, **f32)
        lb = torch.empty(B, n, 3, **i32)
        ub = torch.empty(B, n, 3, **i32)
        nvox = torch.empty(B, n, **i32)
        g2t_offsets = torch.empty(B, n + 1, **i32)
        pws = lib.g2v_batch_plan_workspace(B, n)
        if pws == 0:
            raise RuntimeError(f"batch of {B} scenes x {n} Gaussians exceeds the int32 Gaussian index")
        plan = torch.empty(pws, dtype=torch.uint8, device=dev)
        counts_dev = torch.empty(B + 1, dtype=torch.int64, device=dev)
        # outputs whose size does not depend on the plan's counts, allocated before its host wait
        density = torch.empty(B, X, Y, Z, **f32)
        fdtype = torch.float32 if feats is None else feats.dtype
        fdt = _FEAT_DTYPES[fdtype]
        grid_feats = torch.empty(B, X, Y, Z, C, dtype=fdtype, device=dev)
        start, stop = _timing_events(dev)
        start.record(cur)
        # the (region, Gaussian) pair count of the backward rides on the same launches and wait
        want_bwd = 1 if (keep_t2g and C > 0) else 0
        _lib.check(lib.g2v_batch_forward_plan(B, n, _ptr(means), _ptr(cov), vs, vr, _ptr(cov_inv), _ptr(lb), _ptr(ub),
                                              _ptr(nvox), _ptr(g2t_offsets), _ptr(plan), pws, want_bwd,
                                              _ptr(counts_dev), stream),
                   "gaussian_voxelizer_forward_batched (plan)")
        counts = _pinned_counts(dev, B + 1)
        counts.copy_(counts_dev, non_blocking=True)
        cur.synchronize()   # the one host wait of the batch
        cnt = counts.tolist()
        Ms, MR = [int(v) for v in cnt[:B]], int(cnt[B])
        M = sum(Ms)
        if M > 2147483647 or MR > 2147483647:
            raise RuntimeError(f"batch pair counts {M}, {MR} exceed the int32 CSR")
        g2t_tile_ids = torch.empty(M, **i32)
        ws = torch.empty(lib.g2v_batch_forward_splat_workspace(B, n, C, M, vs, vr), dtype=torch.uint8, device=dev)
        csr = (torch.empty(M, **i32), torch.empty(M, **i32), torch.empty(B * T + 1, **i32)) if keep_t2g \
            else (None, None, None)
        _lib.check(lib.g2v_batch_forward_splat(B, n, C, _ptr(means), _ptr(op), _ptr(feats), fdt, vs, vr, _ptr(cov_inv),
                                               _ptr(lb), _ptr(ub), _ptr(plan), pws, M, _ptr(g2t_tile_ids),
                                               _ptr(density), _ptr(grid_feats), _ptr(csr[0]), _ptr(csr[1]),
                                               _ptr(csr[2]), _ptr(ws), ws.numel(), stream),
                   "gaussian_voxelizer_forward_batched (splat)")
        stop.record(cur)
        batch = None
        if keep_t2g:
            # the backward's outputs and workspace, and its gradient-independent kernels queued
            # behind the forward (after its stop event), as for one scene
            batch = dict(B=B, n=n, C=C, fdt=fdt, M=M, MR=MR, vs=vs, vr=vr, plan=plan, csr=csr, cov_inv=cov_inv,
                         lb=lb, ub=ub, density=density, grid_feats=grid_feats, prepared=False)
            batch["grads"] = (torch.empty(B, n, 3, **f32), torch.empty(B, n, 9, **f32), torch.empty(B, n, **f32),
                              torch.empty(B, n, C, dtype=fdtype, device=dev))
            batch["ws"] = torch.empty(max(1, lib.g2v_batch_backward_workspace(B, n, C, M, MR, vs, vr)),
                                      dtype=torch.uint8, device=dev)
            if C > 0:
                _lib.check(lib.g2v_batch_backward_prepare(B, n, C, vs, vr, _ptr(lb), _ptr(ub), _ptr(feats), fdt, M, MR,
                                                          _ptr(csr[0]), _ptr(csr[1]), _ptr(plan), pws,
                                                          _ptr(batch["ws"]), batch["ws"].numel(), stream),
                           "gaussian_voxelizer_forward_batched (backward preparation)")
                batch["prepared"] = True
        stop.synchronize()
        fwd_sec = start.elapsed_time(stop) / 1000.0
    out, off = [], 0
    for b in range(B):
        out.append((density[b], cov_inv[b], lb[b], ub[b], nvox[b], grid_feats[b], g2t_offsets[b],
                    g2t_tile_ids[off:off + Ms[b]], fwd_sec))
        off += Ms[b]
    return out, density, grid_feats, batch


def _backward_batched(grad_density, grad_feats, means, opacity, features, batch):
    """Backward of _forward_batched(keep_t2g=True): grad_density (B,X,Y,Z), grad_feats (B,X,Y,Z,C)
    (or None: zero); batch = its fourth result.  One g2v_batch_backward call for the B scenes.
    Returns the gradients (B,N,3), (B,N,9), (B,N), (B,N,C) and the time of the batch."""
    lib = _lib.load()
    dev = means.device
    B, n, C, fdt = batch["B"], batch["n"], batch["C"], batch["fdt"]
    gD = _f32_input(grad_density, "grad_density", tuple(batch["density"].shape))
    gF = None
    if C > 0:
        gfeat = batch["grid_feats"]
        gF = grad_feats if grad_feats is not None and grad_feats.shape[-1] > 0 else torch.zeros_like(gfeat)
        if tuple(gF.shape) != tuple(gfeat.shape):
            raise RuntimeError(f"grad_feats_output must be {tuple(gfeat.shape)}, got {tuple(gF.shape)}")
        gF = gF.to(gfeat.dtype).contiguous()
    gm, gc, go, gf = batch["grads"]
    csr, plan = batch["csr"], batch["plan"]
    with _OnDevice(dev):
        cur = torch.cuda.current_stream(dev)
        start, stop = _timing_events(dev)
        start.record(cur)
        _lib.check(lib.g2v_batch_backward(B, n, C, _ptr(gD), _ptr(gF), _ptr(means), _ptr(opacity), _ptr(batch["cov_inv"]),
                                          batch["vs"], batch["vr"], _ptr(batch["lb"]), _ptr(batch["ub"]), batch["M"],
                                          batch["MR"], _ptr(batch["density"]), _ptr(batch["grid_feats"]),
                                          _ptr(features), fdt, _ptr(gm), _ptr(gc), _ptr(go), _ptr(gf), _ptr(csr[0]),
                                          _ptr(csr[1]), _ptr(csr[2]), _ptr(plan), plan.numel(), _ptr(batch["ws"]),
                                          batch["ws"].numel(), 1 if batch["prepared"] else 0,
                                          ctypes.c_void_p(cur.cuda_stream)),
                   "gaussian_voxelizer_backward (batched)")
        stop.record(cur)
        stop.synchronize()
        bwd_sec = start.elapsed_time(stop) / 1000.0
    return gm, gc, go, gf, bwd_sec


def build_t2g(voxel_size, voxel_range, valid_voxel_lb, valid_voxel_ub, g2t_offsets, g2t_tile_ids):
    """The Tile->Gaussian CSR of a forward's G->T pairs (the stable sort of g2t_tile_ids by tile), for
    inspection and parity tests.

    Returns a dict: sorted_tiles (M,), sorted_gauss (M,), tile_offsets (T+1,), and the run-length
    encoding unique_tiles (U,), counts (U,), runs_offsets (U+1,), num_runs.
    """
    lib = _lib.load()
    dev = g2t_offsets.device
    n = g2t_offsets.numel() - 1
    M = g2t_tile_ids.numel()
    vs, vr = _lib.floats(_host_values(voxel_size, 3, "voxel_size")), _lib.floats(_host_values(voxel_range, 6, "voxel_range"))
    (_, tiles) = grid_dims(list(vs), list(vr))
    T = tiles[0] * tiles[1] * tiles[2]
    with torch.cuda.device(dev):
        i32 = dict(dtype=torch.int32, device=dev)
        out = dict(sorted_tiles=torch.empty(M, **i32), sorted_gauss=torch.empty(M, **i32),
                   tile_offsets=torch.empty(T + 1, **i32), unique_tiles=torch.empty(T, **i32),
                   counts=torch.empty(T, **i32), runs_offsets=torch.empty(T + 1, **i32),
                   num_runs=torch.empty(1, **i32))
        ws = torch.empty(lib.g2v_t2g_workspace(n, M, vs, vr), dtype=torch.uint8, device=dev)
        _lib.check(lib.g2v_build_t2g(n, vs, vr, _ptr(valid_voxel_lb), _ptr(valid_voxel_ub),
                                     _ptr(g2t_offsets), _ptr(g2t_tile_ids), M, _ptr(out["sorted_tiles"]),
                                     _ptr(out["sorted_gauss"]), _ptr(out["tile_offsets"]),
                                     _ptr(out["unique_tiles"]), _ptr(out["counts"]),
                                     _ptr(out["runs_offsets"]), _ptr(out["num_runs"]), _ptr(ws),
                                     ws.numel(), _stream(dev)),
                   "build_t2g")
        U = int(out["num_runs"].item())
    out["num_runs"] = U
    out["unique_tiles"] = out["unique_tiles"][:U]
    out["counts"] = out["counts"][:U]
    out["runs_offsets"] = out["runs_offsets"][:U + 1]
    return out


def _cosine_inputs(voxel_label, occ_gt_mask_camera, grid_feats, pseudo_dino_gt):
    """The reference's input checks (src/cuda_feats_loss.cu:158-161: dtype, contiguity, device; a
    failure is a RuntimeError) plus the shape agreement its 3-D / 4-D accessors assume.  grid_feats
    may also be bfloat16 (as the voxelizer returns it for bfloat16 features); pseudo_dino_gt then
    has to be bfloat16 too."""
    fdtype = grid_feats.dtype if isinstance(grid_feats, torch.Tensor) and grid_feats.dtype in _FEAT_DTYPES \
        else torch.float32
    for t, name, dt in ((voxel_label, "voxel_label", torch.float32),
                        (occ_gt_mask_camera, "occ_gt_mask_camera", torch.bool),
                        (grid_feats, "grid_feats", fdtype),
                        (pseudo_dino_gt, "pseudo_dino_gt", fdtype)):
        if not isinstance(t, torch.Tensor) or t.dtype != dt or not t.is_contiguous() or t.device.type != "cuda":
            raise RuntimeError(f"{name} must be a contiguous {dt} GPU tensor")
    if voxel_label.dim() != 3 or grid_feats.dim() != 4:
        raise RuntimeError("voxel_label must be (X, Y, Z) and grid_feats (X, Y, Z, C)")
    dims = tuple(voxel_label.shape)
    if (tuple(occ_gt_mask_camera.shape) != dims or tuple(grid_feats.shape[:3]) != dims
            or tuple(pseudo_dino_gt.shape) != tuple(grid_feats.shape)):
        raise RuntimeError(f"shape mismatch: voxel_label {dims}, occ_gt_mask_camera "
                           f"{tuple(occ_gt_mask_camera.shape)}, grid_feats {tuple(grid_feats.shape)}, "
                           f"pseudo_dino_gt {tuple(pseudo_dino_gt.shape)}")
    dev = grid_feats.device
    for t, name in ((voxel_label, "voxel_label"), (occ_gt_mask_camera, "occ_gt_mask_camera"),
                    (pseudo_dino_gt, "pseudo_dino_gt")):
        if t.device != dev:
            raise RuntimeError(f"{name} is on {t.device}, grid_feats on {dev}")
    return voxel_label.numel(), grid_feats.shape[3], dev, _FEAT_DTYPES[fdtype]


def CudaFeatsCosinelossForward(voxel_label, occ_gt_mask_camera, grid_feats, pseudo_dino_gt):
    """Voxel-wise cosine loss (reference src/cuda_feats_loss.cu:154-231, bound at src/bindings.cpp:67-83).

    Args: voxel_label (X,Y,Z) float32, occ_gt_mask_camera (X,Y,Z) bool, grid_feats and
    pseudo_dino_gt (X,Y,Z,C) float32 (or both bfloat16), all contiguous on the GPU.
    Returns the reference's 3-tuple: the mean over valid voxels (mask and label > 0) of
    1 - cos(grid_feats, pseudo_dino_gt) as a 0-dim GPU tensor (0 without valid voxels), the number
    of valid voxels (int) and the forward time in seconds.
    """
    loss, cnt, fwd_sec, _ = _cosine_forward(voxel_label, occ_gt_mask_camera, grid_feats, pseudo_dino_gt, False)
    return loss, cnt, fwd_sec


def _cosine_forward(voxel_label, occ_gt_mask_camera, grid_feats, pseudo_dino_gt, want_coef):
    """CudaFeatsCosinelossForward; want_coef also returns the (X*Y*Z, 2) float32 tensor of the
    voxels' unscaled gradient coefficients (g2v_cosine_loss_forward_coef), else None."""
    lib = _lib.load()
    V, C, dev, fdt = _cosine_inputs(voxel_label, occ_gt_mask_camera, grid_feats, pseudo_dino_gt)
    with _OnDevice(dev):
        cur = torch.cuda.current_stream(dev)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        cnt_dev = torch.empty((), dtype=torch.int32, device=dev)
        ws = torch.empty(lib.g2v_cosine_loss_workspace(V, C), dtype=torch.uint8, device=dev)
        coef = torch.empty(V, 2, dtype=torch.float32, device=dev) if want_coef else None
        cnt = ctypes.c_int(0)
        start, stop = _timing_events(dev)
        start.record(cur)
        args = (V, C, _ptr(voxel_label), _ptr(occ_gt_mask_camera), _ptr(grid_feats), _ptr(pseudo_dino_gt), fdt,
                _ptr(loss), _ptr(cnt_dev), ctypes.byref(cnt))
        tail = (_ptr(ws), ws.numel(), ctypes.c_void_p(cur.cuda_stream))
        if want_coef:
            _lib.check(lib.g2v_cosine_loss_forward_coef(*args, _ptr(coef), *tail), "CudaFeatsCosinelossForward")
        else:
            _lib.check(lib.g2v_cosine_loss_forward(*args, *tail), "CudaFeatsCosinelossForward")
        stop.record(cur)
        stop.synchronize()
        fwd_sec = start.elapsed_time(stop) / 1000.0
    return loss, int(cnt.value), fwd_sec, coef


def CudaFeatsCosinelossBackward(grad_output, voxel_label, occ_gt_mask_camera, grid_feats, pseudo_dino_gt,
                                num_valid_voxel):
    """Gradient of the cosine loss with respect to grid_feats (reference src/cuda_feats_loss.cu:311-366,
    bound at src/bindings.cpp:85-104).

    grad_output is the upstream gradient of the scalar loss (one element); it is read on the GPU,
    without the reference's host round trip.  Returns (grad_grid_feats (X,Y,Z,C), backward time in
    seconds); the gradient is zero on invalid voxels and has grid_feats' type (a bfloat16 gradient is
    the float value rounded to nearest even).
    """
    lib = _lib.load()
    V, C, dev, fdt = _cosine_inputs(voxel_label, occ_gt_mask_camera, grid_feats, pseudo_dino_gt)
    if not isinstance(grad_output, torch.Tensor) or grad_output.numel() != 1:
        raise RuntimeError("grad_output must be a one-element tensor")
    with _OnDevice(dev):
        cur = torch.cuda.current_stream(dev)
        gout = grad_output.detach().to(device=dev, dtype=torch.float32).reshape(1).contiguous()
        grad_p = torch.empty_like(grid_feats)
        start, stop = _timing_events(dev)
        start.record(cur)
        _lib.check(lib.g2v_cosine_loss_backward(V, C, _ptr(gout), _ptr(voxel_label), _ptr(occ_gt_mask_camera),
                                                _ptr(grid_feats), _ptr(pseudo_dino_gt), fdt, int(num_valid_voxel),
                                                _ptr(grad_p), ctypes.c_void_p(cur.cuda_stream)),
                   "CudaFeatsCosinelossBackward")
        stop.record(cur)
        stop.synchronize()
        bwd_sec = start.elapsed_time(stop) / 1000.0
    return grad_p, bwd_sec


def _scale_rot_inputs(scales, rotations):
    sc = _f32_input(scales, "scales")
    if sc.dim() < 1 or sc.shape[-1] != 3:
        raise RuntimeError(f"scales must be (N, 3), got {tuple(sc.shape)}")
    n = sc.numel() // 3
    rot = _f32_input(rotations, "rotations")
    if tuple(rot.shape) != tuple(sc.shape[:-1]) + (4,):
        raise RuntimeError(f"rotations must be (N, 4) matching scales {tuple(sc.shape)}, got {tuple(rot.shape)}")
    if rot.device != sc.device:
        raise RuntimeError(f"rotations are on {rot.device}, scales on {sc.device}")
    return sc.reshape(-1, 3), rot.reshape(-1, 4), n


def covariance_from_scale_rotation(scales, rotations):
    """Covariances (N, 9) row-major from scales (N, 3) and rotation quaternions (N, 4, real part
    first, normalised here): (R diag(s)) (R diag(s))^T, as ShelfGaussian builds them before the
    voxelizer (reference test/gaussian_voxelizer.py:14-37)."""
    lib = _lib.load()
    sc, rot, n = _scale_rot_inputs(scales, rotations)
    dev = sc.device
    with _OnDevice(dev):
        cov = torch.empty(n, 9, dtype=torch.float32, device=dev)
        _lib.check(lib.g2v_covariance_from_scale_rotation(n, _ptr(sc), _ptr(rot), _ptr(cov), _stream(dev)),
                   "covariance_from_scale_rotation")
    return cov


def covariance_from_scale_rotation_backward(scales, rotations, grad_cov):
    """(grad_scales (N, 3), grad_rotations (N, 4)) for grad_cov (N, 9) = dL/dcovariances."""
    lib = _lib.load()
    sc, rot, n = _scale_rot_inputs(scales, rotations)
    dev = sc.device
    g = _f32_input(grad_cov, "grad_cov")
    if g.numel() != 9 * n:
        raise RuntimeError(f"grad_cov must have N x 9 = {9 * n} elements, got {g.numel()}")
    if g.device != dev:
        raise RuntimeError(f"grad_cov is on {g.device}, scales on {dev}")
    with _OnDevice(dev):
        gs = torch.empty(n, 3, dtype=torch.float32, device=dev)
        gq = torch.empty(n, 4, dtype=torch.float32, device=dev)
        _lib.check(lib.g2v_covariance_from_scale_rotation_backward(n, _ptr(sc), _ptr(rot), _ptr(g), _ptr(gs),
                                                                   _ptr(gq), _stream(dev)),
                   "covariance_from_scale_rotation_backward")
    return gs, gq


# ---- attention in front of the splat --------------------------------------------------------------
# These calls are short, and a training step makes them from two threads (autograd runs backwards on its own), so their
# host side is kept to one check a tensor: checked arguments serve the backward as they are.

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_of(device):
    """The caller's current stream, as a number."""
    if _raw_stream is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _heads_input(t, name, like=None):
    """(B, N, H, D) rows of float32 or bfloat16 on the GPU, in any layout with unit stride along D (others are
    copied); like: the tensor whose type and device it has to share."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a GPU tensor, got {t.device}")
    if t.dtype not in _FEAT_DTYPES:
        raise RuntimeError(f"expected scalar type Float or BFloat16 for {name} but found {t.dtype}")
    if t.dim() != 4:
        raise RuntimeError(f"{name} must be (B, N, H, D), got {tuple(t.shape)}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise RuntimeError(f"{name} is {t.dtype} on {t.device}, expected {like.dtype} on {like.device}")
    return t if t.stride(3) == 1 else t.detach().contiguous()


_Strides = ctypes.c_longlong * 3


def _strides(t):
    return None if t is None else _Strides(*t.stride()[:3])


def _addr(t):
    return None if t is None else t.data_ptr()


def _plain_f32(t, name, shape, device):
    """A contiguous float32 tensor of this shape on this device (None passes)."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != device or t.shape != shape:
        got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise RuntimeError(f"{name} must be float32 {shape} on {device}, got {got}")
    return t if t.is_contiguous() else t.detach().contiguous()


@functools.lru_cache(maxsize=256)
def _workspace_bytes(query, *args):
    """What a *_workspace entry point of the library answers to these sizes (0: refused, by the call itself)."""
    return max(1, getattr(_lib.load(), query)(*args))


def _qk_norm_inputs(q, k, positions, freqs, q_weight, k_weight, k_positions, eps):
    """((q, k, positions, freqs, q_weight, k_weight, k_positions) as the kernels take them, what else a call takes)."""
    q = _heads_input(q, "q")
    B, nq, hq, D = q.shape
    dev = q.device
    nk = hk = 0
    if k is not None:
        k = _heads_input(k, "k", q)
        Bk, nk, hk, Dk = k.shape
        if Bk != B or Dk != D or (k_positions is None and nk != nq):
            raise RuntimeError(f"k {tuple(k.shape)} does not go with q {tuple(q.shape)}"
                               + ("" if k_positions is not None else " (without k_positions the tokens are the same)"))
    else:
        k_positions = k_weight = None
        nk = nq
    if not isinstance(freqs, torch.Tensor) or freqs.dim() != 2:
        raise RuntimeError("freqs must be (axes, pairs)")
    axes, pairs = freqs.shape
    freqs = _plain_f32(freqs, "freqs", (axes, pairs), dev)
    if positions is None:
        raise RuntimeError("positions must be a tensor")
    positions = _plain_f32(positions, "positions", (B, nq, axes), dev)
    k_positions = _plain_f32(k_positions, "k_positions", (B, nk, axes), dev)
    q_weight = _plain_f32(q_weight, "q_weight", (D,), dev)
    k_weight = _plain_f32(k_weight, "k_weight", (D,), dev)
    call = ((B, nq, nk, hq, hk, D, axes), pairs, _FEAT_DTYPES[q.dtype], float(eps))
    return (q, k, positions, freqs, q_weight, k_weight, k_positions), call


def _empty_rows(t):
    """A contiguous tensor like t (a microsecond less of host time than naming shape, type and device)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _qk_norm_forward(inputs, call):
    q, k, pos, freqs, qw, kw, kpos = inputs
    sizes, pairs, fdt, eps = call
    dev = q.device
    with _OnDevice(dev):
        oq = _empty_rows(q)
        ok = None if k is None else _empty_rows(k)
        rc = _lib.load().g2v_qk_norm_rotary_forward(*sizes, pairs, _addr(q), _strides(q), _addr(k), _strides(k), fdt,
                                                    _addr(qw), _addr(kw), _addr(pos), _addr(kpos), _addr(freqs), eps,
                                                    _addr(oq), _addr(ok), _stream_of(dev))
    if rc:
        _lib.check(rc, "qk_norm_rotary_forward")
    return oq, ok


def _qk_norm_backward(gq, gk, inputs, call, want_weights, want_positions):
    q, k, pos, freqs, qw, kw, kpos = inputs
    sizes, pairs, fdt, eps = call
    dev, f32 = q.device, torch.float32
    if gq.shape != q.shape or (k is not None and gk.shape != k.shape):
        raise RuntimeError(f"gradients must be {tuple(q.shape)}" + ("" if k is None else f" and {tuple(k.shape)}"))
    with _OnDevice(dev):
        dq = _empty_rows(q)
        dk = None if k is None else _empty_rows(k)
        dqw = torch.empty(sizes[5], dtype=f32, device=dev) if want_weights[0] else None
        dkw = torch.empty(sizes[5], dtype=f32, device=dev) if want_weights[1] and k is not None else None
        dpos = torch.empty(pos.shape, dtype=f32, device=dev) if want_positions[0] else None
        dkpos = torch.empty(kpos.shape, dtype=f32, device=dev) if want_positions[1] and kpos is not None else None
        nws = _workspace_bytes("g2v_qk_norm_rotary_backward_workspace", *sizes, fdt, 1 if kpos is None else 0)
        ws = torch.empty(nws, dtype=torch.uint8, device=dev)
        rc = _lib.load().g2v_qk_norm_rotary_backward(*sizes, pairs, _addr(q), _strides(q), _addr(k), _strides(k), fdt,
                                                     _addr(qw), _addr(kw), _addr(pos), _addr(kpos), _addr(freqs), eps,
                                                     _addr(gq), _strides(gq), _addr(gk), _strides(gk), _addr(dq),
                                                     _addr(dk), _addr(dqw), _addr(dkw), _addr(dpos), _addr(dkpos),
                                                     ws.data_ptr(), nws, _stream_of(dev))
    if rc:
        _lib.check(rc, "qk_norm_rotary_backward")
    return dq, dk, dqw, dkw, dpos, dkpos


def qk_norm_rotary_forward(q, k, positions, freqs, q_weight=None, k_weight=None, k_positions=None, eps=1e-6):
    """(q', k'): the root-mean-square norm of every head of q (B, Nq, Hq, D) and k (B, Nk, Hk, D; or None), times
    q_weight / k_weight (D,), and its rotation by the token's position: pair i of a head turns by the angle
    sum_a positions[..., a] freqs[a, i].  k_positions None: the keys are the queries' tokens."""
    return _qk_norm_forward(*_qk_norm_inputs(q, k, positions, freqs, q_weight, k_weight, k_positions, eps))


def qk_norm_rotary_backward(grad_q_out, grad_k_out, q, k, positions, freqs, q_weight=None, k_weight=None,
                            k_positions=None, eps=1e-6, want_weights=(True, True), want_positions=(True, True)):
    """(grad_q, grad_k, grad_q_weight, grad_k_weight, grad_positions, grad_k_positions) of qk_norm_rotary_forward; the
    float32 weight and position gradients are None where not wanted (grad_k_positions also with shared positions,
    whose gradient is grad_positions)."""
    inputs, call = _qk_norm_inputs(q, k, positions, freqs, q_weight, k_weight, k_positions, eps)
    gq = _heads_input(grad_q_out, "grad_q_out", inputs[0])
    gk = None if k is None else _heads_input(grad_k_out, "grad_k_out", inputs[0])
    return _qk_norm_backward(gq, gk, inputs, call, want_weights, want_positions)


def _in_place(*tensors):
    """Whether the kernels read these rows where they are (include/g2v.h: in_place)."""
    for t in tensors:
        a, b, c, _ = t.stride()
        if t.dtype != torch.bfloat16 or (a | b | c | t.shape[3]) % 8 or t.data_ptr() % 16 or not 0 <= b < 1 << 24:
            return 0
    return 1


def _attention_inputs(q, k, v, key_mask, scale):
    """((q, k, v, key_mask) as the kernels take them, what else a call takes)."""
    q = _heads_input(q, "q")
    k, v = _heads_input(k, "k", q), _heads_input(v, "v", q)
    B, nq, hq, D = q.shape
    Bk, nk, hk, Dk = k.shape
    if k.shape != v.shape or Bk != B or Dk != D:
        raise RuntimeError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not go with q {tuple(q.shape)}")
    if key_mask is not None:
        if not isinstance(key_mask, torch.Tensor) or key_mask.dtype != torch.bool or key_mask.device != q.device \
                or key_mask.shape != (B, nk):
            raise RuntimeError(f"key_mask must be a bool tensor {(B, nk)} on {q.device}")
        key_mask = key_mask.contiguous()
    return (q, k, v, key_mask), ((B, nq, nk, hq, hk, D), _FEAT_DTYPES[q.dtype], float(D ** -0.5 if scale is None else scale))


def _attention_forward(inputs, call, for_backward):
    q, k, v, key_mask = inputs
    sizes, fdt, scale = call
    B, nq, nk, hq = sizes[:4]
    dev = q.device
    with _OnDevice(dev):
        out = _empty_rows(q)
        rest = _empty_rows(q) if for_backward and fdt == _lib.G2V_DTYPE_BF16 else None
        lse = torch.empty(B, hq, nq, dtype=torch.float32, device=dev) if for_backward else None
        lst = None if key_mask is None else torch.empty(B * (nk + 1), dtype=torch.int32, device=dev)
        nws = _workspace_bytes("g2v_attention_forward_workspace", *sizes, fdt, _in_place(q, k, v), 0 if lst is None else 1)
        ws = torch.empty(nws, dtype=torch.uint8, device=dev)
        rc = _lib.load().g2v_attention_forward(*sizes, _addr(q), _strides(q), _addr(k), _strides(k), _addr(v), _strides(v),
                                               fdt, _addr(key_mask), scale, _addr(out), _addr(rest), _addr(lse), _addr(lst),
                                               ws.data_ptr(), nws, _stream_of(dev))
    if rc:
        _lib.check(rc, "attention_forward")
    return out, rest, lse, lst


def _attention_backward(g, q, k, v, out, rest, lse, key_list, call, want_q, want_kv):
    sizes, fdt, scale = call
    dev = q.device
    if g.shape != q.shape:
        raise RuntimeError(f"grad_out must be {tuple(q.shape)}, got {tuple(g.shape)}")
    with _OnDevice(dev):
        dq = _empty_rows(q) if want_q else None
        dk = _empty_rows(k) if want_kv else None
        dv = _empty_rows(k) if want_kv else None
        nws = _workspace_bytes("g2v_attention_backward_workspace", *sizes, fdt, _in_place(q, k, v, g),
                               0 if key_list is None else 1)
        ws = torch.empty(nws, dtype=torch.uint8, device=dev)
        rc = _lib.load().g2v_attention_backward(*sizes, _addr(q), _strides(q), _addr(k), _strides(k), _addr(v), _strides(v),
                                                fdt, _addr(key_list), scale, _addr(out), _addr(rest), _addr(lse), _addr(g),
                                                _strides(g), _addr(dq), _addr(dk), _addr(dv), ws.data_ptr(), nws,
                                                _stream_of(dev))
    if rc:
        _lib.check(rc, "attention_backward")
    return dq, dk, dv


def attention_forward(q, k, v, key_mask=None, scale=None, for_backward=False):
    """(out, rest, lse, key_list): softmax(scale q k^T over the valid keys) v for q (B, Nq, Hq, D) and k, v (B, Nk, Hkv, D),
    Hq a multiple of Hkv; scale None: D^-1/2.  key_mask (B, Nk) bool, False where a key is not attended to.  rest (what
    rounding took from a bfloat16 out) and lse, None unless for_backward, and key_list, None without a mask, are what
    attention_backward takes."""
    return _attention_forward(*_attention_inputs(q, k, v, key_mask, scale), for_backward)


def attention_backward(grad_out, q, k, v, out, rest, lse, key_list=None, scale=None, want_q=True, want_kv=True):
    """(grad_q, grad_k, grad_v) of attention_forward from its results; None where not wanted."""
    (q, k, v, _), call = _attention_inputs(q, k, v, None, scale)
    B, nq, nk, hq = call[0][:4]
    dev = q.device
    g = _heads_input(grad_out, "grad_out", q)
    _check_saved(out, "out", q.dtype, dev)
    _check_saved(lse, "lse", torch.float32, dev)
    if rest is not None:
        _check_saved(rest, "rest", torch.bfloat16, dev)
        if rest.shape != out.shape:
            raise RuntimeError(f"rest must be {tuple(out.shape)}, got {tuple(rest.shape)}")
    if out.shape != q.shape or lse.shape != (B, hq, nq):
        raise RuntimeError(f"out {tuple(out.shape)} and lse {tuple(lse.shape)} do not go with q {tuple(q.shape)}")
    if key_list is not None:
        _check_saved(key_list, "key_list", torch.int32, dev)
        if key_list.numel() != B * (nk + 1):
            raise RuntimeError(f"key_list must hold {B * (nk + 1)} values, got {key_list.numel()}")
    return _attention_backward(g, q, k, v, out, rest, lse, key_list, call, want_q, want_kv)


# ---- attention within a window ----------------------------------------------------------------------

@functools.lru_cache(maxsize=256, typed=True)
def _window_bounds(left, right, sinks):
    """(left, right, sinks) as the library takes them: places, -1 without a bound."""
    for side, name in ((left, "left"), (right, "right")):
        if side is not None and (isinstance(side, bool) or not isinstance(side, int) or side < 0):
            raise RuntimeError(f"window: {name} must be a number of places or None, got {side!r}")
    if isinstance(sinks, bool) or not isinstance(sinks, int) or sinks < 0:
        raise RuntimeError(f"sinks must be a number of keys, got {sinks!r}")
    return tuple(-1 if side is None else min(side, 1 << 30) for side in (left, right)) + (min(sinks, 1 << 30),)


def _window(window, sinks):
    if not isinstance(window, (tuple, list)) or len(window) != 2:
        raise RuntimeError(f"window must be (left, right), got {window!r}")
    return _window_bounds(window[0], window[1], sinks)


def _window_attention_forward(inputs, call, window, for_backward):
    q, k, v, key_mask = inputs
    sizes, fdt, scale = call
    B, nq, nk, hq = sizes[:4]
    dev = q.device
    with _OnDevice(dev):
        out = _empty_rows(q)
        rest = _empty_rows(q) if for_backward and fdt == _lib.G2V_DTYPE_BF16 else None
        lse = torch.empty(B, hq, nq, dtype=torch.float32, device=dev) if for_backward else None
        nws = _workspace_bytes("g2v_window_attention_forward_workspace", *sizes, fdt, *window, _in_place(q, k, v),
                               0 if key_mask is None else 1)
        ws = torch.empty(nws, dtype=torch.uint8, device=dev)
        rc = _lib.load().g2v_window_attention_forward(*sizes, _addr(q), _strides(q), _addr(k), _strides(k), _addr(v), _strides(v),
                                                      fdt, _addr(key_mask), *window, scale, _addr(out), _addr(rest), _addr(lse),
                                                      ws.data_ptr(), nws, _stream_of(dev))
    if rc:
        _lib.check(rc, "window_attention_forward")
    return out, rest, lse


def _window_attention_backward(g, q, k, v, key_mask, out, rest, lse, call, window, want_q, want_kv):
    sizes, fdt, scale = call
    dev = q.device
    if g.shape != q.shape:
        raise RuntimeError(f"grad_out must be {tuple(q.shape)}, got {tuple(g.shape)}")
    with _OnDevice(dev):
        dq = _empty_rows(q) if want_q else None
        dk = _empty_rows(k) if want_kv else None
        dv = _empty_rows(k) if want_kv else None
        nws = _workspace_bytes("g2v_window_attention_backward_workspace", *sizes, fdt, *window, _in_place(q, k, v, g),
                               0 if key_mask is None else 1)
        ws = torch.empty(nws, dtype=torch.uint8, device=dev)
        rc = _lib.load().g2v_window_attention_backward(*sizes, _addr(q), _strides(q), _addr(k), _strides(k), _addr(v),
                                                       _strides(v), fdt, _addr(key_mask), *window, scale, _addr(out),
                                                       _addr(rest), _addr(lse), _addr(g), _strides(g), _addr(dq), _addr(dk),
                                                       _addr(dv), ws.data_ptr(), nws, _stream_of(dev))
    if rc:
        _lib.check(rc, "window_attention_backward")
    return dq, dk, dv


def window_attention_forward(q, k, v, window, sinks=0, key_mask=None, scale=None, for_backward=False):
    """(out, rest, lse): attention_forward over the keys that each query sees.  Query i stands at key place p = i + Nk - Nq and
    sees key j if j <= p + right and (j >= p - left or j < sinks), with window = (left, right), None for no bound.  rest and lse,
    None unless for_backward, are what window_attention_backward takes."""
    return _window_attention_forward(*_attention_inputs(q, k, v, key_mask, scale), _window(window, sinks), for_backward)


def window_attention_backward(grad_out, q, k, v, out, rest, lse, window, sinks=0, key_mask=None, scale=None, want_q=True,
                              want_kv=True):
    """(grad_q, grad_k, grad_v) of window_attention_forward from its results; None where not wanted."""
    (q, k, v, key_mask), call = _attention_inputs(q, k, v, key_mask, scale)
    B, nq, _, hq = call[0][:4]
    dev = q.device
    g = _heads_input(grad_out, "grad_out", q)
    _check_saved(out, "out", q.dtype, dev)
    _check_saved(lse, "lse", torch.float32, dev)
    if rest is not None:
        _check_saved(rest, "rest", torch.bfloat16, dev)
        if rest.shape != out.shape:
            raise RuntimeError(f"rest must be {tuple(out.shape)}, got {tuple(rest.shape)}")
    if out.shape != q.shape or lse.shape != (B, hq, nq):
        raise RuntimeError(f"out {tuple(out.shape)} and lse {tuple(lse.shape)} do not go with q {tuple(q.shape)}")
    return _window_attention_backward(g, q, k, v, key_mask, out, rest, lse, call, _window(window, sinks), want_q, want_kv)


# ---- layer norm --------------------------------------------------------------------------------------

def _rows_input(t, name, like=None):
    """(rows as (B, N, C) with unit stride along C, their strides along B and N); like: the tensor whose type, device and shape it
    has to share.  Leading dimensions are taken together where their strides allow it, others are copied."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a GPU tensor, got {t.device}")
    if t.dtype not in _FEAT_DTYPES:
        raise RuntimeError(f"expected scalar type Float or BFloat16 for {name} but found {t.dtype}")
    if t.dim() < 1:
        raise RuntimeError(f"{name} must be (..., C), got a scalar")
    if like is not None and (t.dtype != like.dtype or t.device != like.device or t.shape != like.shape):
        raise RuntimeError(f"{name} is {t.dtype} {tuple(t.shape)} on {t.device}, expected {like.dtype} {tuple(like.shape)} on "
                           f"{like.device}")
    C = t.shape[-1]
    if C and t.numel() // C >= 1 << 31:
        raise RuntimeError(f"{name} has {t.numel() // C} rows (limit 2^31)")
    if t.is_contiguous():
        n = t.numel() // C if C else 0
        return t, (1, n, C), (n * C, C)
    if t.dim() == 3 and t.stride(2) == 1:
        return t, tuple(t.shape), t.stride()[:2]
    if t.dim() == 2 and t.stride(1) == 1:
        return t, (1,) + tuple(t.shape), (0, t.stride(0))
    return _rows_input(t.detach().contiguous(), name)


_RowStrides = ctypes.c_longlong * 2


def _row_strides(rows):
    return None if rows is None else _RowStrides(*rows[2])


def _norm_weight(t, name, C, device, like=None):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype not in _FEAT_DTYPES or t.device != device or t.shape != (C,):
        got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise RuntimeError(f"{name} must be float32 or bfloat16 {(C,)} on {device}, got {got}")
    if like is not None and t.dtype != like.dtype:
        raise RuntimeError(f"{name} is {t.dtype}, weight {like.dtype}")
    return t if t.is_contiguous() else t.detach().contiguous()


def _same_rows(rows, other):
    """Two inputs' rows with one split of their leading dimensions (that of the one that is not contiguous)."""
    if rows[1] == other[1]:
        return rows, other
    if rows[1][0] == 1 and rows[0].is_contiguous():
        B, n, C = other[1]
        return (rows[0], other[1], (n * C, C)), other
    if other[1][0] == 1 and other[0].is_contiguous():
        return _same_rows(other, rows)[::-1]
    return _same_rows(rows, _rows_input(other[0].detach().contiguous(), "rows"))


def layer_norm_forward(x, weight=None, bias=None, residual=None, eps=1e-5, for_backward=False):
    """(y, sum, stats): the layer norm of the rows of x (..., C), or of sum = x + residual, with weight and bias (C,).  sum is None
    without residual; stats, None unless for_backward, holds the rows' mean and (variance + eps)^-1/2 for layer_norm_backward."""
    rows, other = _rows_input(x, "x"), None
    if residual is not None:
        rows, other = _same_rows(rows, _rows_input(residual, "residual", x))
    C, dev = x.shape[-1], x.device
    weight = _norm_weight(weight, "weight", C, dev)
    bias = _norm_weight(bias, "bias", C, dev, weight)
    wdt = next((_FEAT_DTYPES[t.dtype] for t in (weight, bias) if t is not None), _lib.G2V_DTYPE_F32)
    with _OnDevice(dev):
        y = _empty_rows(x)
        total = None if residual is None else _empty_rows(x)
        stats = torch.empty(x.numel() // C if C else 0, 2, dtype=torch.float32, device=dev) if for_backward else None
        rc = _lib.load().g2v_layer_norm_forward(*rows[1], rows[0].data_ptr(), _row_strides(rows),
                                                None if other is None else other[0].data_ptr(), _row_strides(other),
                                                _FEAT_DTYPES[x.dtype], _addr(weight), _addr(bias), wdt, float(eps), y.data_ptr(),
                                                _addr(total), _addr(stats), _stream_of(dev))
    if rc:
        _lib.check(rc, "layer_norm_forward")
    return y, total, stats


def layer_norm_backward(grad_y, x, weight, stats, grad_sum=None, want_weights=(True, True), bias_dtype=None):
    """(grad_x, grad_weight, grad_bias) of layer_norm_forward from what it normed (x, or the sum with the residual, whose gradient is
    grad_x as well) and its stats; grad_sum: the gradient that reaches the sum besides.  Weight gradients have the weight's type
    (without one bias_dtype, None: float32) and are None where not wanted."""
    rows, gy = _rows_input(x, "x"), _rows_input(grad_y, "grad_y", x)
    C, dev = x.shape[-1], x.device
    weight = _norm_weight(weight, "weight", C, dev)
    _check_saved(stats, "stats", torch.float32, dev)
    if stats.shape != (x.numel() // C if C else 0, 2):
        raise RuntimeError(f"stats {tuple(stats.shape)} do not go with x {tuple(x.shape)}")
    rows, gy = _same_rows(rows, gy)
    gs = None
    if grad_sum is not None:
        gs = _rows_input(grad_sum, "grad_sum", x)
        if gs[1] != rows[1]:      # three layouts that share no split of the leading dimensions
            rows, gy, gs = (_rows_input(t[0].detach().contiguous(), "rows") for t in (rows, gy, gs))
    wdtype = weight.dtype if weight is not None else bias_dtype or torch.float32
    with _OnDevice(dev):
        dx = _empty_rows(x)
        dw = torch.empty(C, dtype=wdtype, device=dev) if want_weights[0] else None
        db = torch.empty(C, dtype=wdtype, device=dev) if want_weights[1] else None
        nws = _workspace_bytes("g2v_layer_norm_backward_workspace", *rows[1], _FEAT_DTYPES[x.dtype])
        ws = torch.empty(nws, dtype=torch.uint8, device=dev)
        rc = _lib.load().g2v_layer_norm_backward(*rows[1], rows[0].data_ptr(), _row_strides(rows), _FEAT_DTYPES[x.dtype],
                                                 _addr(weight), _FEAT_DTYPES[wdtype], stats.data_ptr(), gy[0].data_ptr(),
                                                 _row_strides(gy), None if gs is None else gs[0].data_ptr(), _row_strides(gs),
                                                 dx.data_ptr(), _addr(dw), _addr(db), ws.data_ptr(), nws, _stream_of(dev))
    if rc:
        _lib.check(rc, "layer_norm_backward")
    return dx, dw, db


# ---- gradient norm and clipping ----------------------------------------------------------------------

def _dense(t):
    """Whether a tensor's elements are one piece of memory, each once, in some order of its dimensions."""
    return t.is_contiguous() or torch.ops.aten.is_non_overlapping_and_dense(t)


def _reaches(target, steps):
    """Whether target is a sum of step x over the (step, most) of steps, 0 <= x <= most: the largest step first, whose x the others' reach
    and divisor leave few values (one or two where strides nest).  Also True where 10,000 looks do not tell."""
    merged = {}
    for step, most in steps:
        if step and most > 0:
            merged[step] = merged.get(step, 0) + most
    order = sorted(merged.items(), reverse=True)
    reach, divisor = [0], [0]    # of the steps behind each
    for step, most in reversed(order):
        reach.append(reach[-1] + step * most)
        divisor.append(math.gcd(divisor[-1], step))
    reach.reverse()
    divisor.reverse()
    looks = 0
    todo = [(0, target)]
    while todo:
        k, left = todo.pop()
        if left == 0:
            return True
        if left < 0 or left > reach[k] or left % divisor[k]:
            continue
        step, most = order[k]
        lo, hi = max(0, -((reach[k + 1] - left) // step)), min(most, left // step)
        looks += hi - lo + 1
        if looks > 10000:
            return True
        todo.extend((k + 1, left - step * x) for x in range(lo, hi + 1))
    return False


def _byte_steps(t):
    size = t.element_size()
    return [(step * size, n - 1) for step, n in zip(t.stride(), t.shape)]


def _reach_of(t):
    """Bytes from a tensor's first element to its last one's end."""
    return sum(step * most for step, most in _byte_steps(t)) + t.element_size()


def _share_memory(t, o):
    """Whether two tensors with elements have bytes in common: t + i = o + j for bytes i and j of theirs, j taken from its end."""
    return _reaches(o.data_ptr() - t.data_ptr() + _reach_of(o) - 1,
                    _byte_steps(t) + _byte_steps(o) + [(1, t.element_size() - 1), (1, o.element_size() - 1)])


def _overlaps_itself(t):
    """Whether two elements of a tensor have one place: the first dimension whose indexes differ, by one at least, and those behind it, by
    anything, make up for each other."""
    steps = sorted((step, n) for step, n in zip(t.stride(), t.shape) if n > 1)
    reach = 0
    for step, n in steps:
        if step <= reach:
            break
        reach += step * (n - 1)
    else:    # every step is beyond what the smaller ones reach
        return False
    return any(_reaches(sum(s * (m - 1) for s, m in steps[k + 1:]) - step, [(step, n - 2)] + [(s, 2 * (m - 1)) for s, m in steps[k + 1:]])
               for k, (step, n) in enumerate(steps))


def _same_places(t, o):
    """Whether two tensors of one shape have each element at the same place and of the same type."""
    return t.data_ptr() == o.data_ptr() and t.dtype == o.dtype \
        and all(a == b or n == 1 for a, b, n in zip(t.stride(), o.stride(), t.shape))


def _check_sharing(grads, outs):
    """Refuses what the library refuses among flat tensors, whose memory it sees: an output that shares memory with another one, or with a
    gradient but for its own at the same places, and with itself."""
    spans = [(t.data_ptr(), t.data_ptr() + _reach_of(t), i, t, written) for written, tensors in ((True, outs), (False, grads))
             for i, t in enumerate(tensors) if t.numel() and (written or t is not outs[i])]
    spans.sort(key=lambda span: span[0])
    open_ = []
    for at, end, i, t, written in spans:
        if written and _overlaps_itself(t):
            raise RuntimeError(f"clip_gradients: elements of tensor {i}, which is written, share memory")
        open_ = [span for span in open_ if span[1] > at]
        for _, _, k, o, other in open_:
            if (written or other) and not (i == k and _same_places(t, o)) and _share_memory(t, o):
                raise RuntimeError(f"clip_gradients: tensors {min(i, k)} and {max(i, k)} share memory that is written")
        open_.append((at, end, i, t, written))


def _clip_checked(grads, outs, dev):
    """(gradients, outputs, results to copy back) as flat memory: tensors of other layouts go through contiguous copies."""
    for i, (g, o) in enumerate(zip(grads, outs)):
        for t, what in ((g, "gradient"), (o, "output")):
            if t.device != dev or t.layout != torch.strided or t.dtype not in _FEAT_DTYPES or t.shape != g.shape:
                raise RuntimeError(f"{what} {i} must be float32 or bfloat16 {tuple(g.shape)} on {dev}, got {t.dtype} "
                                   f"{tuple(t.shape)} ({t.layout}) on {t.device}")
    flat = [g.stride() == o.stride() and _dense(g) for g, o in zip(grads, outs)]
    if not all(flat):    # the library sees the copies' memory
        _check_sharing(grads, outs)
    src, dst, back = [], [], []
    for g, o, as_is in zip(grads, outs, flat):
        if not as_is:
            same = o is g
            g = g.contiguous()
            if same or not o.is_contiguous():
                back.append((o, g if same else torch.empty(o.shape, dtype=o.dtype, device=dev)))
                o = back[-1][1]
        src.append(g)
        dst.append(o)
    return src, dst, back


_tensor_dtype, _tensor_shape = operator.attrgetter("dtype"), operator.attrgetter("shape")


def clip_gradients(grads, max_norm, outs=None):
    """The norm (a 0-dim float32 GPU tensor) of a list of gradient tensors taken together, float32 or bfloat16 on one GPU; each is
    scaled by min(1, max_norm / (norm + 1e-6)), in place or into outs, tensors of the same shapes (float32 or bfloat16)."""
    lib = _lib.load()
    if not grads:
        raise RuntimeError("clip_gradients: no tensors")
    dev = grads[0].device
    if dev.type != "cuda":
        raise RuntimeError(f"gradients must be GPU tensors, got {dev}")
    if outs is not None and len(outs) != len(grads):
        raise RuntimeError(f"{len(grads)} gradients, but {len(outs)} outputs")
    into = grads if outs is None else outs
    # a model's hundreds of tensors are looked over by a few passes, half a microsecond each; whatever is out of line is named by
    # the slower way
    T, src, dst, back = torch.Tensor, grads, into, ()
    types = list(map(_tensor_dtype, grads))
    into_types = types if outs is None else list(map(_tensor_dtype, outs))
    plain = {*types, *into_types} <= _FEAT_DTYPES.keys() and set(map(T.get_device, grads)) == {dev.index} \
        and all(map(T.is_contiguous, grads))
    if plain and outs is not None:
        plain = set(map(T.get_device, outs)) == {dev.index} and all(map(T.is_contiguous, outs)) \
            and list(map(_tensor_shape, grads)) == list(map(_tensor_shape, outs))
    if not plain:
        src, dst, back = _clip_checked(grads, into, dev)

    def arrays(tensors, types):
        return array.array("Q", map(T.data_ptr, tensors)), array.array("i", map(_FEAT_DTYPES.__getitem__, types))

    with _OnDevice(dev):
        n = len(src)
        numels = array.array("q", map(T.numel, src))
        gp, gd = arrays(src, types)
        op, od = (gp, gd) if dst is src else arrays(dst, into_types)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        nws = _workspace_bytes("g2v_clip_gradients_workspace", n)
        ws = torch.empty(nws, dtype=torch.uint8, device=dev)
        rc = lib.g2v_clip_gradients(n, gp.buffer_info()[0], gd.buffer_info()[0], op.buffer_info()[0], od.buffer_info()[0],
                                    numels.buffer_info()[0], float(max_norm), norm.data_ptr(), ws.data_ptr(), nws, _stream_of(dev))
        if rc:
            _lib.check(rc, "clip_gradients")
        for t, result in back:
            t.copy_(result)
    torch.autograd.graph.increment_version(into)
    return norm
