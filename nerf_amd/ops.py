"""Tensor-level wrappers over the C ABI: torch tensors in, torch tensors out, on the current HIP
stream.  Shape checks live here (the kernels trust their arguments); arithmetic lives in the
library.  Nothing in this module computes on the CPU."""
import ctypes

import numpy as np
import torch

from . import _native as nv


def _dev(t=None):
    if t is not None and isinstance(t, torch.Tensor) and t.is_cuda:
        return t.device
    if not torch.cuda.is_available():
        raise nv.NerfHipError("no GPU visible: nerf_amd runs on MI355X only (there is no CPU path)")
    return torch.device("cuda", torch.cuda.current_device())


def get_rays(H, W, focal, c2w):
    """run_nerf_helpers.py:122-129 -> rays_o, rays_d as [H,W,3] fp32 tensors."""
    dev = _dev(c2w if isinstance(c2w, torch.Tensor) else None)
    m = np.ascontiguousarray(torch.as_tensor(c2w).detach().cpu().numpy()[:3, :4], dtype=np.float32)
    rays_o = torch.empty((int(H), int(W), 3), dtype=torch.float32, device=dev)
    rays_d = torch.empty_like(rays_o)
    with torch.cuda.device(dev):
        nv.check(nv.lib().nerf_get_rays(int(H), int(W), float(focal),
                                        m.ctypes.data_as(ctypes.c_void_p), nv.ptr(rays_o),
                                        nv.ptr(rays_d), nv.stream()), "nerf_get_rays")
    return rays_o, rays_d


def ndc_rays(H, W, focal, near, rays_o, rays_d):
    """run_nerf_helpers.py:145-180 on [...,3] tensors."""
    o = nv.f32(rays_o)
    d = nv.f32(rays_d, o.device)
    if o.shape != d.shape or o.shape[-1] != 3:
        raise ValueError(f"ndc_rays: rays_o {tuple(o.shape)} and rays_d {tuple(d.shape)} must both be [...,3]")
    oo, od = torch.empty_like(o), torch.empty_like(d)
    with torch.cuda.device(o.device):
        nv.check(nv.lib().nerf_ndc_rays(o.numel() // 3, int(H), int(W), float(focal), float(near),
                                        nv.ptr(o), nv.ptr(d), nv.ptr(oo), nv.ptr(od), nv.stream()),
                 "nerf_ndc_rays")
    return oo, od


def build_ray_batch(rays_o, rays_d, view_src, ndc, H, W, focal, near, far):
    """render()'s assembly of the [N, 8|11] ray batch (run_nerf.py:79-108).
    near/far: python scalars or per-ray tensors [N] / [N,1]."""
    o = nv.f32(rays_o).reshape(-1, 3)
    d = nv.f32(rays_d, o.device).reshape(-1, 3)
    n = o.shape[0]
    if d.shape[0] != n:
        raise ValueError("build_ray_batch: rays_o and rays_d disagree on the ray count")
    v = None
    if view_src is not None:
        v = nv.f32(view_src, o.device).reshape(-1, 3)
        if v.shape[0] != n:
            raise ValueError("build_ray_batch: view directions disagree on the ray count")
    width = 11 if v is not None else 8
    near_t = far_t = None
    near_s = far_s = 0.0
    if isinstance(near, (torch.Tensor, np.ndarray)) and isinstance(far, (torch.Tensor, np.ndarray)):
        near_t = nv.f32(near, o.device).reshape(-1)
        far_t = nv.f32(far, o.device).reshape(-1)
        if near_t.numel() != n or far_t.numel() != n:
            raise ValueError("build_ray_batch: per-ray near/far must have one value per ray")
    else:
        near_s, far_s = float(near), float(far)
    out = torch.empty((n, width), dtype=torch.float32, device=o.device)
    with torch.cuda.device(o.device):
        nv.check(nv.lib().nerf_build_ray_batch(n, nv.ptr(o), nv.ptr(d), nv.ptr(v), int(bool(ndc)),
                                               int(H), int(W), float(focal), nv.ptr(near_t),
                                               nv.ptr(far_t), near_s, far_s, nv.ptr(out), width,
                                               nv.stream()), "nerf_build_ray_batch")
    return out


def gather_pixel_rays(H, W, focal, poses, images, img_index, pix_index):
    """(batch_rays [2,n,3], target [n,3] or None) for pixels pix_index (row*W+col) of images img_index.
    poses [n_img,3,4] fp32 and images [n_img,H,W,C>=3] fp32 (or None) live on the GPU."""
    poses = nv.f32(poses)
    dev = poses.device
    if poses.dim() != 3 or tuple(poses.shape[1:]) != (3, 4):
        raise ValueError(f"gather_pixel_rays: poses must be [n_img,3,4], got {tuple(poses.shape)}")
    n_img = poses.shape[0]
    channels = 0
    if images is not None:
        images = nv.f32(images, dev)
        if images.dim() != 4 or tuple(images.shape[:3]) != (n_img, H, W) or images.shape[3] < 3:
            raise ValueError(f"gather_pixel_rays: images must be [{n_img},{H},{W},>=3], got {tuple(images.shape)}")
        channels = images.shape[3]
    ii = torch.as_tensor(img_index, device=dev).to(torch.int32).contiguous().reshape(-1)
    pi = torch.as_tensor(pix_index, device=dev).to(torch.int32).contiguous().reshape(-1)
    if ii.shape != pi.shape:
        raise ValueError("gather_pixel_rays: img_index and pix_index differ in length")
    n = ii.numel()
    rays = torch.empty((2, n, 3), dtype=torch.float32, device=dev)
    rgb = torch.empty((n, 3), dtype=torch.float32, device=dev) if images is not None else None
    if n == 0:
        return rays, rgb
    with torch.cuda.device(dev):
        nv.check(nv.lib().nerf_gather_pixel_rays(int(H), int(W), float(focal), n_img, nv.ptr(poses), nv.ptr(images),
                                                 channels, nv.ptr(ii), nv.ptr(pi), n, nv.ptr(rays), nv.ptr(rgb),
                                                 nv.stream()), "nerf_gather_pixel_rays")
    return rays, rgb


def embed(x, L):
    """Embedder.embed (run_nerf_helpers.py:22-56) on [...,3] -> [..., 3+6L]."""
    x = nv.f32(x)
    if x.shape[-1] != 3:
        raise ValueError("embed: last dimension must be 3")
    out = torch.empty(tuple(x.shape[:-1]) + (3 + 6 * L,), dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        nv.check(nv.lib().nerf_embed(x.numel() // 3, nv.ptr(x), int(L), nv.ptr(out), nv.stream()),
                 "nerf_embed")
    return out


def sample_z(rays, S, lindisp=False, perturb_u=None):
    """Stratified depths [N,S] for a ray batch [N,width>=8]."""
    rays = nv.f32(rays)
    n, width = rays.shape
    u = None
    if perturb_u is not None:
        u = nv.f32(perturb_u, rays.device)
        if tuple(u.shape) != (n, S):
            raise ValueError(f"sample_z: perturb_u must be [{n},{S}]")
    z = torch.empty((n, S), dtype=torch.float32, device=rays.device)
    with torch.cuda.device(rays.device):
        nv.check(nv.lib().nerf_sample_z(n, int(S), nv.ptr(rays), width, int(bool(lindisp)),
                                        nv.ptr(u), nv.ptr(z), nv.stream()), "nerf_sample_z")
    return z


# When a list, every MLP launch appends (start_event, end_event, points) -- bench.py's roofline leg.
MLP_TIMING = None


# When a dict, the compositing and resampling launches append (start_event, end_event,
# algorithmic bytes) under their kernel's name -- bench.py's HBM-bound kernels.
HBM_TIMING = None


def _timed_hbm(name, nbytes, launch):
    if HBM_TIMING is None:
        return launch()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    launch()
    e1.record()
    HBM_TIMING.setdefault(name, []).append((e0, e1, nbytes))


def _timed_mlp(points, launch):
    if MLP_TIMING is None:
        return launch()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    launch()
    e1.record()
    MLP_TIMING.append((e0, e1, points))


def packed_bytes():
    return int(nv.lib().nerf_mlp_packed_bytes())


def mlp_pack(params, packed):
    """params: 24 contiguous fp32 CUDA tensors in get_weights() order; packed: uint8 [packed_bytes()]."""
    arr = (ctypes.c_void_p * 24)(*[p.data_ptr() for p in params])
    with torch.cuda.device(packed.device):
        nv.check(nv.lib().nerf_mlp_pack(arr, nv.ptr(packed), nv.stream()), "nerf_mlp_pack")


def mlp_forward_rays(packed, rays, z):
    """raw [N,S,4] for points o + d*z of a ray batch [N,11] with depths z [N,S]."""
    n, width = rays.shape
    S = z.shape[1]
    if z.shape[0] != n:
        raise ValueError("mlp_forward_rays: rays and z disagree on the ray count")
    raw = torch.empty((n, S, 4), dtype=torch.float32, device=rays.device)
    with torch.cuda.device(rays.device):
        _timed_mlp(n * S, lambda: nv.check(
            nv.lib().nerf_mlp_forward_rays(nv.ptr(packed), nv.ptr(rays), width, nv.ptr(z), n, S,
                                           nv.ptr(raw), nv.stream()), "nerf_mlp_forward_rays"))
    return raw


def mlp_forward_pts(packed, pts, viewdirs):
    """raw [N,S,4] for explicit points [N,S,3] and per-ray view directions [N,3]."""
    n, S = pts.shape[0], pts.shape[1]
    if tuple(viewdirs.shape) != (n, 3) or pts.shape[2] != 3:
        raise ValueError("mlp_forward_pts: need pts [N,S,3] and viewdirs [N,3]")
    raw = torch.empty((n, S, 4), dtype=torch.float32, device=pts.device)
    with torch.cuda.device(pts.device):
        _timed_mlp(n * S, lambda: nv.check(
            nv.lib().nerf_mlp_forward_pts(nv.ptr(packed), nv.ptr(pts), nv.ptr(viewdirs), n, S,
                                          nv.ptr(raw), nv.stream()), "nerf_mlp_forward_pts"))
    return raw


def composite_fwd(raw, z, rays_d, d_stride, white_bkgd=False, noise=None, noise_std=0.0,
                  want_weights=True):
    """raw2outputs.  rays_d is any fp32 tensor whose row i starts the direction of ray i when read
    with stride d_stride (e.g. the ray batch offset by 3 columns)."""
    n, S = z.shape
    dev = z.device
    rgb = torch.empty((n, 3), dtype=torch.float32, device=dev)
    disp = torch.empty((n,), dtype=torch.float32, device=dev)
    acc = torch.empty((n,), dtype=torch.float32, device=dev)
    depth = torch.empty((n,), dtype=torch.float32, device=dev)
    weights = torch.empty((n, S), dtype=torch.float32, device=dev) if want_weights else None
    with torch.cuda.device(dev):
        # algorithmic bytes: raw 16 S + z 4 S + direction 12 read, weights 4 S + maps 24 written
        _timed_hbm(f"composite_fwd S={S}", n * (24 * S + 36), lambda: nv.check(
            nv.lib().nerf_composite_fwd(nv.ptr(raw), nv.ptr(z), ctypes.c_void_p(rays_d.data_ptr()),
                                        int(d_stride), n, S, int(bool(white_bkgd)),
                                        nv.ptr(noise), float(noise_std), nv.ptr(rgb),
                                        nv.ptr(disp), nv.ptr(acc), nv.ptr(depth),
                                        nv.ptr(weights), nv.stream()), "nerf_composite_fwd"))
    return rgb, disp, acc, weights, depth


def sample_pdf(bins, weights, N_samples, det=False, u=None):
    """run_nerf_helpers.py:185-213 on [...,nb] bins and [...,nb-1] weights."""
    bins = nv.f32(bins)
    weights = nv.f32(weights, bins.device)
    nb = bins.shape[-1]
    if weights.shape[-1] != nb - 1 or weights.shape[:-1] != bins.shape[:-1]:
        raise ValueError(f"sample_pdf: bins {tuple(bins.shape)} need weights [..., {nb - 1}]")
    lead = tuple(bins.shape[:-1])
    n = bins.numel() // nb
    if not det:
        if u is None:
            u = torch.rand(lead + (N_samples,), dtype=torch.float32, device=bins.device)
        u = nv.f32(u, bins.device)
        if tuple(u.shape) != lead + (N_samples,):
            raise ValueError("sample_pdf: u must be [..., N_samples]")
    else:
        u = None
    out = torch.empty(lead + (N_samples,), dtype=torch.float32, device=bins.device)
    with torch.cuda.device(bins.device):
        nv.check(nv.lib().nerf_sample_pdf(nv.ptr(bins), nv.ptr(weights), n, nb, int(N_samples),
                                          int(bool(det)), nv.ptr(u), nv.ptr(out), nv.stream()),
                 "nerf_sample_pdf")
    return out


def resample_merge(z_vals, weights, N_importance, det=True, u=None, want_samples=True):
    """z_mid -> sample_pdf(weights[:,1:-1]) -> sort(concat) of render_rays, one kernel.
    Returns z_fine [N,Sc+Si], z_samples [N,Si] (or None), z_std [N]."""
    n, Sc = z_vals.shape
    dev = z_vals.device
    if tuple(weights.shape) != (n, Sc):
        raise ValueError("resample_merge: weights must match z_vals")
    if not det:
        if u is None:
            u = torch.rand((n, N_importance), dtype=torch.float32, device=dev)
        u = nv.f32(u, dev)
        if tuple(u.shape) != (n, N_importance):
            raise ValueError("resample_merge: u must be [N, N_importance]")
    else:
        u = None
    z_out = torch.empty((n, Sc + N_importance), dtype=torch.float32, device=dev)
    z_samples = torch.empty((n, N_importance), dtype=torch.float32, device=dev) if want_samples else None
    z_std = torch.empty((n,), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        # algorithmic bytes: z and weights read (8 Sc), merged depths written (4 (Sc + Si))
        _timed_hbm(f"resample_merge {Sc}+{N_importance}", n * (8 * Sc + 4 * (Sc + N_importance)), lambda: nv.check(
            nv.lib().nerf_resample_merge(nv.ptr(z_vals), nv.ptr(weights), n, Sc,
                                         int(N_importance), int(bool(det)), nv.ptr(u),
                                         nv.ptr(z_out), nv.ptr(z_samples), nv.ptr(z_std),
                                         nv.stream()), "nerf_resample_merge"))
    return z_out, z_samples, z_std


# (device, stream) -> grow-only workspace of render_rays_single_call.  One per stream: calls on
# different streams of one GPU may overlap and must not share intermediates; a workspace that is
# outgrown is only dropped by the stream that used it, behind the work that stream has queued.
_RENDER_WS = {}


def render_rays_single_call(packed_coarse, packed_fine, rays, N_samples, N_importance, lindisp=False,
                            white_bkgd=False, perturb_u=None, pdf_u=None):
    """The whole per-ray core through ONE call of the C ABI (nerf_render_rays).  Returns the dict
    render_rays returns at raw_noise_std = 0 without `raw`."""
    n, width = rays.shape
    dev = rays.device
    need = int(nv.lib().nerf_render_rays_workspace_bytes(n, int(N_samples), int(N_importance)))
    key = (dev, torch.cuda.current_stream(dev).cuda_stream)
    ws = _RENDER_WS.get(key)
    if ws is None or ws.numel() < need:
        ws = _RENDER_WS[key] = torch.empty((max(need, 1),), dtype=torch.uint8, device=dev)
        ws.record_stream(torch.cuda.current_stream(dev))
    new = lambda *shape: torch.empty(shape, dtype=torch.float32, device=dev)
    ret = dict(rgb_map=new(n, 3), disp_map=new(n), acc_map=new(n), depth_map=new(n))
    if N_importance > 0:
        ret.update(rgb0=new(n, 3), disp0=new(n), acc0=new(n), z_std=new(n))
    g = lambda k: nv.ptr(ret.get(k))
    with torch.cuda.device(dev):
        nv.check(nv.lib().nerf_render_rays(nv.ptr(packed_coarse), nv.ptr(packed_fine), nv.ptr(rays), width, n,
                                           int(N_samples), int(N_importance), int(bool(lindisp)), int(bool(white_bkgd)),
                                           nv.ptr(perturb_u), nv.ptr(pdf_u), g('rgb_map'), g('disp_map'), g('acc_map'),
                                           g('depth_map'), g('rgb0'), g('disp0'), g('acc0'), g('z_std'), nv.ptr(ws),
                                           nv.stream()), "nerf_render_rays")
    return ret


def composite_bwd(raw, z, rays_d, d_stride, white_bkgd, noise, noise_std, g_rgb, g_acc=None, g_depth=None):
    """d_raw [N,S,4] from the gradients of rgb_map / acc_map / depth_map (None = zero)."""
    n, S = z.shape
    d_raw = torch.empty((n, S, 4), dtype=torch.float32, device=z.device)
    with torch.cuda.device(z.device):
        nv.check(nv.lib().nerf_composite_bwd(nv.ptr(raw), nv.ptr(z), ctypes.c_void_p(rays_d.data_ptr()),
                                             int(d_stride), n, S, int(bool(white_bkgd)), nv.ptr(noise),
                                             float(noise_std), nv.ptr(g_rgb), nv.ptr(g_acc),
                                             nv.ptr(g_depth), nv.ptr(d_raw), nv.stream()),
                 "nerf_composite_bwd")
    return d_raw


def act_bytes(n_points):
    return int(nv.lib().nerf_mlp_act_bytes(int(n_points)))


def train_layout():
    """Block numbers of the saved training tensors (nerf_mlp_train_layout), as a dict."""
    out = (ctypes.c_int32 * 10)()
    nv.check(nv.lib().nerf_mlp_train_layout(out, 10), "nerf_mlp_train_layout")
    names = ("act_blocks", "pe", "h0", "v", "vpe", "mask", "grad_blocks", "d_v", "d_pre0", "d_alpha")
    return dict(zip(names, (int(x) for x in out)))


def mlp_forward_train(packed, rays, z, act):
    """mlp_forward_rays that also fills `act` (uint8 [act_bytes(N*S)]) for the backward pass."""
    n, width = rays.shape
    S = z.shape[1]
    raw = torch.empty((n, S, 4), dtype=torch.float32, device=rays.device)
    if act.numel() < act_bytes(n * S):
        raise ValueError("mlp_forward_train: activation scratch too small")
    with torch.cuda.device(rays.device):
        _timed_mlp(n * S, lambda: nv.check(
            nv.lib().nerf_mlp_forward_train(nv.ptr(packed), nv.ptr(rays), width, nv.ptr(z), n, S,
                                            nv.ptr(raw), nv.ptr(act), nv.stream()), "nerf_mlp_forward_train"))
    return raw


def packed_bwd_bytes():
    return int(nv.lib().nerf_mlp_packed_bwd_bytes())


def mlp_pack_bwd(params, packed_bwd):
    arr = (ctypes.c_void_p * 24)(*[p.data_ptr() for p in params])
    with torch.cuda.device(packed_bwd.device):
        nv.check(nv.lib().nerf_mlp_pack_bwd(arr, nv.ptr(packed_bwd), nv.stream()), "nerf_mlp_pack_bwd")


def grad_bytes(n_points):
    return int(nv.lib().nerf_mlp_grad_bytes(int(n_points)))


def partial_bytes():
    return int(nv.lib().nerf_mlp_partial_bytes())


GRAD_SATURATED, GRAD_UNDERFLOW = 1, 2


def mlp_backward_status(partial):
    """(flags, gscale_used, max|d_raw|) of the last mlp_backward that used `partial`; waits for it."""
    flags, gs, mx = ctypes.c_int(0), ctypes.c_float(0.), ctypes.c_float(0.)
    with torch.cuda.device(partial.device):
        nv.check(nv.lib().nerf_mlp_backward_status(nv.ptr(partial), ctypes.byref(flags), ctypes.byref(gs),
                                                   ctypes.byref(mx), nv.stream()), "nerf_mlp_backward_status")
    return flags.value, gs.value, mx.value


def mlp_backward(packed_bwd, act, d_raw, gscale, gbuf, partial, grads, accumulate=False):
    """Parameter gradients (24 tensors shaped like the parameters, written in place) from
    d_raw [N,S,4] and the activations saved by mlp_forward_train.  gscale None or 0: the fp16
    gradient scale is formed on the device from max|d_raw| (largest scaled element in [256, 512));
    gscale < 0: the same with the target [-gscale, -2 gscale), a power of two; > 0: used as given."""
    gscale = 0.0 if gscale is None else gscale
    n_points = d_raw.numel() // 4
    if gbuf.numel() < grad_bytes(n_points) or partial.numel() < partial_bytes():
        raise ValueError("mlp_backward: scratch too small")
    arr = (ctypes.c_void_p * 24)(*[g.data_ptr() for g in grads])
    with torch.cuda.device(d_raw.device):
        nv.check(nv.lib().nerf_mlp_backward(nv.ptr(packed_bwd), nv.ptr(act), nv.ptr(d_raw), n_points,
                                            float(gscale), nv.ptr(gbuf), nv.ptr(partial), arr,
                                            int(bool(accumulate)), nv.stream()), "nerf_mlp_backward")


# ---- dense layers in 8 bits -------------------------------------------------------------------------
# One layer y = relu(x W + b) of a network that is queried or trained layer by layer (any widths): its
# input rows are held in 8-bit integers with a scale per row, which the product reads and which is all
# that is kept for the backward pass; its weights in 8-bit integers with a scale per output channel.
#
#     w8 = pack_int8(W, pow2=True)                                   # whenever W changes
#     rows = quantize_rows(x, pow2=True, want_mask=True)
#     y = linear_int8(rows, w8, b, relu=True, dtype=torch.bfloat16)  # or linear_int8_quantized: y in 8 bits
#     dW, db = linear_int8_grad_weight(rows, dz)                     # dz = gradient before this layer's ReLU
#     dx = linear_int8_grad_input(dz, w8, rows.mask)                 # ... before the ReLU that made x
#
# Gradients are those of the product of the 8-bit numbers; rounding to 8 bits passes them on unchanged.
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _padded_width(k):
    return -(-int(k) // 64) * 64


def _on_gpu(what, *tensors):
    """All given tensors on one GPU -> its device."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{what}: expected tensors, got {type(t).__name__}")
        if not t.is_cuda:
            raise nv.NerfHipError(f"{what}: expected a tensor on the GPU (the HIP path has no CPU fallback)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"{what}: tensors on {dev} and {t.device}")
    return dev


_ENTRY = {}   # name -> entry point of the library


def _call(name, dev, *args):
    """One entry point on `dev` and its current stream; device pointers as integers.  (A call for one ray is
    all host time: no context manager and no stream object where the device is the current one.)"""
    fn = _ENTRY.get(name)
    if fn is None:
        fn = _ENTRY[name] = getattr(nv.lib(), name)
    index = dev.index
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        nv.check(rc, name)


def _addr(t):
    return None if t is None else t.data_ptr()


def _row_major(what, t, width=None):
    """(tensor, row distance) of a [n, k] tensor of one of the three types whose rows are runs in memory;
    a tensor with any other strides is copied."""
    if t.dim() != 2 or t.shape[1] < 1 or (width is not None and t.shape[1] != width):
        raise ValueError(f"{what}: expected [n, {'k >= 1' if width is None else width}], got {tuple(t.shape)}")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{what}: expected float32, float16 or bfloat16, got {t.dtype}")
    n, k = t.shape
    if (k > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < k):
        t = t.contiguous()
    return t, (max(t.stride(0), k) if n > 1 else k)


class Int8Rows:
    """Rows in 8-bit integers: q [n, k rounded up to 64] int8 with zeros behind column k, scale [n] fp32 (an
    element is q * scale); pow2: the scales are powers of two (what gradients ask for); mask: None, or
    the bits x > 0 of the rows as [n, width of q / 8] uint8 (bit f & 7 of byte f >> 3)."""

    __slots__ = ("q", "scale", "k", "pow2", "mask")

    def __init__(self, q, scale, k, pow2=False, mask=None):
        _on_gpu("Int8Rows", q, scale, mask)
        k = int(k)
        if q.dtype != torch.int8 or q.dim() != 2 or k < 1 or q.shape[1] != _padded_width(k):
            raise ValueError(f"Int8Rows: q must be int8 [n, {_padded_width(k)}] for k = {k}, got {q.dtype} {tuple(q.shape)}")
        if scale.dtype != torch.float32 or tuple(scale.shape) != (q.shape[0],):
            raise ValueError(f"Int8Rows: scale must be float32 [{q.shape[0]}], got {scale.dtype} {tuple(scale.shape)}")
        if mask is not None and (mask.dtype != torch.uint8 or tuple(mask.shape) != (q.shape[0], q.shape[1] // 8)):
            raise ValueError(f"Int8Rows: mask must be uint8 [{q.shape[0]}, {q.shape[1] // 8}], got {mask.dtype} {tuple(mask.shape)}")
        if not (q.is_contiguous() and scale.is_contiguous() and (mask is None or mask.is_contiguous())):
            raise ValueError("Int8Rows: expected contiguous tensors")
        self.q, self.scale, self.k, self.pow2, self.mask = q, scale, k, bool(pow2), mask

    @classmethod
    def _made(cls, q, scale, k, pow2, mask):
        """Of tensors that _new_rows made."""
        self = cls.__new__(cls)
        self.q, self.scale, self.k, self.pow2, self.mask = q, scale, k, bool(pow2), mask
        return self

    @property
    def n(self):
        return self.q.shape[0]

    def __repr__(self):
        return f"Int8Rows(n={self.n}, k={self.k}, pow2={self.pow2}, mask={'yes' if self.mask is not None else 'no'})"


class Int8Weights:
    """What pack_int8 returns: the integers and channel scales of W [k, m] as the kernels read them."""

    __slots__ = ("packed", "k", "m", "pow2")

    def __init__(self, packed, k, m, pow2):
        need = nv.lib().nerf_int8_packed_bytes(int(k), int(m), 1 if pow2 else 0)
        if need == 0 or packed.dtype != torch.uint8 or tuple(packed.shape) != (need,) or not packed.is_contiguous():
            raise ValueError(f"Int8Weights: packed must be {need} contiguous bytes for {k} x {m}, got {packed.dtype} {tuple(packed.shape)}")
        self.packed, self.k, self.m, self.pow2 = packed, int(k), int(m), bool(pow2)

    def __repr__(self):
        return f"Int8Weights(k={self.k}, m={self.m}, pow2={self.pow2})"


def _new(shape, dtype, dev):
    # (the cheapest of torch's allocations from Python)
    return torch.empty_strided(shape, (shape[1], 1) if len(shape) == 2 else (1,), dtype=dtype, device=dev)


def _new_rows(n, k, dev, want_mask):
    kp = _padded_width(k)
    return (_new((n, kp), torch.int8, dev), _new((n,), torch.float32, dev),
            _new((n, kp // 8), torch.uint8, dev) if want_mask else None)


def quantize_rows(x, pow2=False, want_mask=False):
    """Int8Rows of x [n, k] (float32, float16 or bfloat16): one scale per row, max|x| / 127 or, with pow2, the
    next power of two (up to twice the step; rows that a gradient is taken through need it)."""
    dev = _on_gpu("quantize_rows", x)
    x, ld = _row_major("quantize_rows", x)
    n, k = x.shape
    q, scale, mask = _new_rows(n, k, dev, want_mask)
    _call("nerf_quantize_rows", dev, x.data_ptr(), _DTYPES[x.dtype], n, k, ld, 1 if pow2 else 0, q.data_ptr(), scale.data_ptr(),
          _addr(mask))
    return Int8Rows._made(q, scale, k, pow2, mask)


def pack_int8(w, pow2=False, into=None):
    """Int8Weights of a kernel W [k, m] (fp32, [in, out]): one scale per output channel.  pow2 also lays out
    what linear_int8_grad_input reads.  into: Int8Weights of the same shape and kind whose memory is
    overwritten (behind the work that the current stream has queued)."""
    dev = _on_gpu("pack_int8", w)
    if w.dim() != 2 or w.shape[0] < 1 or w.shape[1] < 1:
        raise ValueError(f"pack_int8: expected [k >= 1, m >= 1], got {tuple(w.shape)}")
    if w.dtype != torch.float32 or not w.is_contiguous():
        w = nv.f32(w.detach(), dev)
    k, m = w.shape
    need = nv.lib().nerf_int8_packed_bytes(k, m, 1 if pow2 else 0)
    if need == 0:
        raise ValueError(f"pack_int8: widths {k} x {m} are beyond what the kernels are built for")
    if into is None:
        packed = _new((need,), torch.uint8, dev)
    elif not isinstance(into, Int8Weights) or (into.k, into.m, into.pow2, into.packed.device) != (k, m, bool(pow2), dev):
        raise ValueError(f"pack_int8: into={into!r} does not hold {k} x {m} weights, pow2={bool(pow2)}, on {dev}")
    else:
        packed = into.packed
    _call("nerf_int8_pack", dev, w.data_ptr(), k, m, 1 if pow2 else 0, packed.data_ptr())
    return Int8Weights(packed, k, m, bool(pow2)) if into is None else into


def _linear_inputs(what, rows, weights, bias, addend):
    if not isinstance(rows, Int8Rows) or not isinstance(weights, Int8Weights):
        raise ValueError(f"{what}: expected Int8Rows and Int8Weights")
    dev = _on_gpu(what, rows.q, weights.packed, bias, addend)
    if rows.k != weights.k:
        raise ValueError(f"{what}: rows of {rows.k} elements against weights for {weights.k}")
    if bias is not None:
        if bias.dtype != torch.float32 or not bias.is_contiguous():
            bias = nv.f32(bias.detach(), dev)
        if tuple(bias.shape) != (weights.m,):
            raise ValueError(f"{what}: bias must be [{weights.m}], got {tuple(bias.shape)}")
    ldadd, add_dtype = 0, 0
    if addend is not None:
        addend, ldadd = _row_major(f"{what} (addend)", addend.detach(), weights.m)
        if addend.dtype == torch.float16:  # exact
            addend, ldadd = addend.float(), weights.m
        add_dtype = _DTYPES[addend.dtype]
        if addend.shape[0] != rows.n:
            raise ValueError(f"{what}: addend must have {rows.n} rows, got {addend.shape[0]}")
    return dev, bias, addend, add_dtype, ldadd


def linear_int8(rows, weights, bias=None, relu=False, addend=None, dtype=torch.float32):
    """y [n, m] = x W (+ bias) (+ addend [n, m]), then relu when asked: the product of the 8-bit integers with
    exact sums, scaled and finished in fp32, stored in `dtype`."""
    dev, bias, addend, add_dtype, ldadd = _linear_inputs("linear_int8", rows, weights, bias, addend)
    if dtype not in _DTYPES:
        raise ValueError(f"linear_int8: dtype must be float32, float16 or bfloat16, got {dtype}")
    n, m = rows.n, weights.m
    y = _new((n, m), dtype, dev)
    _call("nerf_linear_int8", dev, rows.q.data_ptr(), rows.scale.data_ptr(), n, rows.k, weights.packed.data_ptr(), m, _addr(bias),
          _addr(addend), add_dtype, ldadd, 1 if relu else 0, y.data_ptr(), _DTYPES[dtype], m)
    return y


def _through_fp32(n, k, m):
    """Whether an 8-bit output of these sizes is faster by way of a stored fp32 row, in two calls.  Device time, one call / two
    calls, us:
     - up to 512 outputs a row is one workgroup's, which walks its inputs step by step: with few rows of many inputs the
       many small workgroups of the product alone are faster, weights in LDS or not.  640 x 64, 2048 rows 10.7 / 9.6, 12288
       rows 11.0 / 11.1; 896 x 128, 8192 rows 14.3 / 13.2; 640 x 256, 8192 rows 17.8 / 14.6, 12288 rows 17.9 / 21.4; 640 x 512,
       4096 rows 18.3 / 15.2, 8192 rows 18.8 / 26.7.  Up to 576 inputs the two are close, and one call is less host time;
     - beyond, the products are formed twice.  With few tiles: 256 x 576, 4096 rows 21.2 / 16.1, 8192 rows 21.9 / 25.2; 512 x
       2048, 2048 rows 29.0 / 23.5, 4096 rows 30.1 / 35.0.  With many inputs: 640 x 1024, 32768 rows 66 / 69, 896 x 1024 79 /
       77, 1024 x 1024 87 / 79; once the fp32 rows do not stay in the 256 MB cache in front of memory: 1024 x 1024, 131072
       rows 317 / 369, 1280 x 1024 369 / 401, 2048 x 2048, 32768 rows 271 / 240."""
    groups = -(-m // 64)
    if m <= 512:
        return k > 576 and n < 12288 and n * groups < 40960
    return n * groups <= 65536 or k > (768 if n * m * 4 <= 256 << 20 else 1280)


def linear_int8_quantized(rows, weights, bias=None, relu=False, addend=None, pow2=False, want_mask=False):
    """quantize_rows(linear_int8(...), pow2, want_mask), with y in fp32 in between: the next layer's input.  One
    call that never stores y, but where storing it is faster or an addend is not a multiple of 64 wide: the two
    calls."""
    dev, bias, addend, add_dtype, ldadd = _linear_inputs("linear_int8_quantized", rows, weights, bias, addend)
    n, m = rows.n, weights.m
    if (addend is not None and m % 64 != 0) or _through_fp32(n, rows.k, m):
        return quantize_rows(linear_int8(rows, weights, bias, relu, addend), pow2, want_mask)
    q, scale, mask = _new_rows(n, m, dev, want_mask)
    need = nv.lib().nerf_linear_int8_quantized_bytes(n, m) if m > 512 else 0
    ws = _new((need,), torch.uint8, dev) if need else None
    _call("nerf_linear_int8_quantized", dev, rows.q.data_ptr(), rows.scale.data_ptr(), n, rows.k, weights.packed.data_ptr(), m,
          _addr(bias), _addr(addend), add_dtype, ldadd, 1 if relu else 0, 1 if pow2 else 0, q.data_ptr(), scale.data_ptr(), _addr(mask),
          _addr(ws), need)
    return Int8Rows._made(q, scale, m, pow2, mask)


def linear_int8_grad_input(dz, weights, mask=None):
    """dx [n, k] = dz [n, m] W^T in dz's type, with W as the forward product used it (packed with pow2); zero
    where `mask` (of the rows that were the layer's input) says that the input was not positive."""
    what = "linear_int8_grad_input"
    if not isinstance(weights, Int8Weights):
        raise ValueError(f"{what}: expected Int8Weights")
    if not weights.pow2:
        raise ValueError(f"{what}: weights must be packed with pow2=True")
    dev = _on_gpu(what, dz, weights.packed, mask)
    dz, ld = _row_major(what, dz, weights.m)
    n = dz.shape[0]
    if mask is not None and not mask.is_contiguous():
        mask = mask.contiguous()
    if mask is not None and (mask.dtype != torch.uint8 or tuple(mask.shape) != (n, _padded_width(weights.k) // 8)):
        raise ValueError(f"{what}: mask must be uint8 [{n}, {_padded_width(weights.k) // 8}], got {mask.dtype} {tuple(mask.shape)}")
    dx = _new((n, weights.k), dz.dtype, dev)
    _call("nerf_linear_int8_grad_input", dev, dz.data_ptr(), _DTYPES[dz.dtype], n, weights.m, ld, weights.packed.data_ptr(), weights.k,
          _addr(mask), dx.data_ptr(), weights.k)
    return dx


def linear_int8_grad_weight(rows, dz):
    """(dW [k, m], db [m]) in fp32 from the rows the forward pass kept (made with pow2) and dz [n, m].  The same
    inputs give the same bits."""
    what = "linear_int8_grad_weight"
    if not isinstance(rows, Int8Rows):
        raise ValueError(f"{what}: expected Int8Rows")
    if not rows.pow2:
        raise ValueError(f"{what}: the rows' scales must be powers of two (quantize_rows(..., pow2=True))")
    dev = _on_gpu(what, rows.q, dz)
    dz, ld = _row_major(what, dz)
    n, m = dz.shape
    if n != rows.n:
        raise ValueError(f"{what}: {rows.n} rows against {n} of dz")
    if n == 0:
        return (torch.zeros((rows.k, m), dtype=torch.float32, device=dev), torch.zeros((m,), dtype=torch.float32, device=dev))
    dw, db = _new((rows.k, m), torch.float32, dev), _new((m,), torch.float32, dev)
    need = nv.lib().nerf_linear_int8_grad_weight_bytes(n, rows.k, m)
    ws = _new((need,), torch.uint8, dev) if need else None
    _call("nerf_linear_int8_grad_weight", dev, rows.q.data_ptr(), rows.scale.data_ptr(), n, rows.k, dz.data_ptr(), _DTYPES[dz.dtype], m,
          ld, dw.data_ptr(), db.data_ptr(), _addr(ws), need)
    return dw, db
