"""The reference's network (run_nerf_helpers.py:80-117) evaluated and trained layer by layer on the 8-bit
dense-layer kernels, for the widths and depths the fused kernels are not built for.

Every layer's input is held in 8-bit integers with one scale per point; a hidden layer reads the integers of the
layer before and leaves its own (ops.linear_int8_quantized: one launch, but for layers wider than 512 and for few
points, where it may be two with an fp32 row in between).  The layers that take an encoding beside the layer before
have one product for each, the encoding's being added in the epilogue of the other.  For the backward pass the
integers, scales and ReLU bits are all that is kept: about 2.8 KB per point of the 8 x 256 network, where the fused
kernels save 4.7 KB.  A query that records nothing keeps one layer at a time and makes no bits.
Gradients between layers are bf16, parameter gradients fp32; rounding to 8 bits passes gradients on
unchanged.

The encoded point is one row, coordinates and sines under one scale, the next power of two of its largest value over
127: the sines' step is 1/64 while every coordinate is below 1.98 in size, 1/32 below 3.97, 1/16 below 7.9.  Scenes are
best scaled to about +-2.  Off the same network in 64 bits (8 x 256, rms, in standard deviations of the density and
colour outputs): 3.5 and 1.8 % with coordinates up to 2, 3.7 and 2.1 % up to 4, 4.1 and 2.3 % up to 6 (with coordinates and
sines apart 3.3 and 2.1 % there: most of it is the layers' own rounding).

    model = init_nerf_model(D=4, W=128, input_ch=63, input_ch_views=27, skips=[2], use_viewdirs=True,
                            precision='int8')
    render_kwargs_train, ... = create_nerf(args)        # args.precision = 'int8'
"""
import torch

from . import _native as nv
from . import ops
from .run_nerf_helpers import LaidOut, NerfModel

# Points evaluated at a time when nothing is recorded: no more than these, and as many as the network's widest layer
# leaves within these bytes of transient memory (256 wide: at most 3.1 GiB for 2^20; 4096 wide: 103 thousand points).
_QUERY_POINTS = 1 << 20
_QUERY_BYTES = 4 << 30


class LayeredNerfModel(NerfModel):
    """A NerfModel of any depth, width, encoding and skips (view directions required) on the 8-bit layers."""

    layered = True

    def __init__(self, D, W, input_ch, input_ch_views, output_ch, skips, use_viewdirs, device=None, generator=None):
        super().__init__(D, W, input_ch, input_ch_views, output_ch, skips, use_viewdirs, device=device, generator=generator)
        self._packed8 = LaidOut(self.device)

    @staticmethod
    def check_shape(D, W, input_ch, input_ch_views, output_ch, skips, use_viewdirs):
        def encoded(n):
            return n >= 3 and (n - 3) % 6 == 0
        if not (use_viewdirs and output_ch == 4 and 1 <= D <= 64 and 2 <= W <= 4096 and encoded(input_ch) and encoded(input_ch_views)
                and all(s >= 0 for s in skips)):  # (one at or behind the last layer has no effect, as in the reference)
            raise NotImplementedError(
                "the layered 8-bit network takes view directions, output_ch=4, depths 1 to 64, widths 2 to 4096 and inputs of "
                f"3 + 6 L values; got D={D} W={W} input_ch={input_ch} input_ch_views={input_ch_views} output_ch={output_ch} "
                f"skips={list(skips)} use_viewdirs={use_viewdirs}")

    # parameters of layer i (Keras order): 0 .. D-1 point layers, then bottleneck, view, rgb, alpha
    def weight(self, i):
        return self.params[2 * i]

    def bias(self, i):
        return self.params[2 * i + 1]

    def split(self, i):
        """Rows of W of layer i that take the encoding, in front (skip layers) or behind (view layer), and
        those that take the layer before: [(first row, rows, is encoding)] in the order of W."""
        k = self.shapes[i][0]
        if i == self.D + 1:
            return [(0, 256, False), (256, self.input_ch_views, True)]
        if i == 0 or i == self.D + 2:
            return [(0, k, i == 0)]
        before = self.D - 1 if i >= self.D else i - 1
        if before in self.skips:
            return [(0, self.input_ch, True), (self.input_ch, k - self.input_ch, False)]
        return [(0, k, False)]

    def packed8(self):
        """Per layer its Int8Weights, one for each part of split(), for the current parameters (re-laid in the
        same memory when they change, also by a captured graph)."""

        def lay(old):
            return [[ops.pack_int8(self.weight(i)[r0:r0 + n], pow2=True, into=old[i][j] if old else None)
                     for j, (r0, n, _) in enumerate(self.split(i))] for i in range(len(self.shapes))]
        return self._packed8.current(self._version(), lay, lambda layers: (w.packed for parts in layers for w in parts))


def _row_bytes(k):
    return -(-k // 64) * 64 + 4


def point_bytes(model):
    """Upper bound of the device memory that a point takes in a pass that records nothing: both encodings (fp32 and 8 bits),
    and of one layer its input rows, its output rows, an addend and an fp32 row (where ops.linear_int8_quantized makes two
    calls), and the four outputs twice."""
    both = model.input_ch, model.input_ch_views
    layer = max(sum(_row_bytes(n) for _, n, _ in model.split(i)) + _row_bytes(m) + 8 * m for i, (_, m) in enumerate(model.shapes))
    return sum(_row_bytes(c) + 4 * c for c in both) + layer + 2 * 16


def query_points(model):
    return max(1, min(_QUERY_POINTS, _QUERY_BYTES // point_bytes(model)))


def _pieces(P, S, most):
    """(first point, one behind the last, first ray, points per ray) of pieces of at most `most` points: whole rays, or parts
    of one where a ray's S points are more than that."""
    if S <= most:
        step = most // S * S
        return [(a, min(a + step, P), a // S, S) for a in range(0, P, step)]
    return [(a, min(a + most, r * S + S), r, min(most, r * S + S - a)) for r in range(P // S) for a in range(r * S, r * S + S, most)]


def _encode(x, channels):
    return ops.embed(x, (channels - 3) // 6) if channels > 3 else x


class _Pass:
    """One forward pass: raw [P, 4], and for gradients() the rows of every layer's input, in the order of split()."""

    def __init__(self, model, pts, viewdirs, S, record=True):
        """pts [P, 3], viewdirs [P / S, 3], all fp32.  record: whether rows and ReLU bits are kept (without, a layer's rows
        go when the next layer's are there, and no bits are made)."""
        self.model = model
        packed = self.packed = model.packed8()
        self.version = model._version()
        D = model.D
        pe = ops.quantize_rows(_encode(pts, model.input_ch), pow2=True)
        # one encoding per ray, its integers repeated for the ray's points
        ve = ops.quantize_rows(_encode(viewdirs, model.input_ch_views), pow2=True)
        ve = ops.Int8Rows(ve.q.repeat_interleave(S, dim=0), ve.scale.repeat_interleave(S), ve.k, pow2=True)
        self.inputs = [None] * len(model.shapes)

        def dense(i, parts, **out):
            # the narrow part of a concatenated input first, as the addend of the other: a partial sum, in fp32 (in bf16 it
            # would save 5 % of a training step and 14 % of a query)
            if record:
                self.inputs[i] = parts
            add = None
            at = [j for j, (_, _, enc) in enumerate(model.split(i)) if not enc or len(parts) == 1][0]
            for j, rows in enumerate(parts):
                if j != at:
                    add = ops.linear_int8(rows, packed[i][j])
            if 'dtype' in out:
                return ops.linear_int8(parts[at], packed[i][at], model.bias(i), addend=add, **out)
            return ops.linear_int8_quantized(parts[at], packed[i][at], model.bias(i), addend=add, pow2=True, **out)

        h = [pe]
        for i in range(D):
            y = dense(i, h, relu=True, want_mask=record)
            h = [pe, y] if i in model.skips else [y]
        alpha = dense(D + 3, h, dtype=torch.float32)
        h = [dense(D, h), ve]
        h = [dense(D + 1, h, relu=True, want_mask=record)]
        rgb = dense(D + 2, h, dtype=torch.float32)
        self.raw = torch.cat([rgb, alpha], dim=1)

    def gradients(self, d_raw):
        """Gradients of the parameters, in their order, from d raw [P, 4] fp32."""
        model, packed, D = self.model, self.packed, self.model.D
        if model._version() != self.version:
            raise RuntimeError("the network's parameters changed between its forward and its backward pass")
        grads = [None] * len(model.params)

        def parameters(i, dz):
            parts = [ops.linear_int8_grad_weight(rows, dz) for rows in self.inputs[i]]
            grads[2 * i] = parts[0][0] if len(parts) == 1 else torch.cat([p[0] for p in parts], dim=0)
            grads[2 * i + 1] = parts[0][1]

        def back(i, dz, mask=True):
            at = [j for j, (_, _, enc) in enumerate(model.split(i)) if not enc][0]
            return ops.linear_int8_grad_input(dz, packed[i][at], self.inputs[i][at].mask if mask else None)

        d16 = d_raw.to(torch.bfloat16)
        parameters(D + 2, d_raw[:, :3])
        dz = back(D + 2, d16[:, :3])                                    # before the view layer's ReLU
        parameters(D + 1, dz)
        dz = back(D + 1, dz, mask=False)                                # the bottleneck is linear
        parameters(D, dz)
        parameters(D + 3, d_raw[:, 3:])
        dz = back(D, dz).add_(back(D + 3, d16[:, 3:]))                  # before the last point layer's ReLU
        for i in range(D - 1, -1, -1):
            parameters(i, dz)
            if i:
                dz = back(i, dz)
        # one flat buffer that the gradients tile: the optimiser and a gradient exchange take it whole
        flat, out, at = torch.cat([g.reshape(-1) for g in grads]), [], 0
        for p in model.params:
            out.append(flat[at:at + p.numel()].view(p.shape))
            at += p.numel()
        return out


def query(model, pts, viewdirs, S):
    """raw [P, 4] of points [P, 3] with one view direction per S points, nothing recorded."""
    P = pts.shape[0]
    if P == 0:
        return pts.new_empty((0, 4))
    pieces = _pieces(P, S, query_points(model))
    with torch.no_grad():
        if len(pieces) == 1:
            return _Pass(model, pts, viewdirs, S, record=False).raw
        out = pts.new_empty((P, 4))
        for a, b, ray, s in pieces:
            out[a:b] = _Pass(model, pts[a:b], viewdirs[ray:ray + (b - a) // s], s, record=False).raw
        return out


class LayeredQuery(torch.autograd.Function):
    """raw = network(rays, z) on the 8-bit layers; backward yields the parameter gradients (none for rays
    and depths, as for the fused network)."""

    @staticmethod
    def forward(ctx, rays, z, model, *params):
        ctx.set_materialize_grads(False)
        n, S = z.shape
        pts = (rays[:, None, 0:3] + rays[:, None, 3:6] * z[:, :, None]).reshape(n * S, 3)
        ctx.run = _Pass(model, pts, rays[:, 8:11].contiguous(), S)
        return ctx.run.raw.view(n, S, 4)

    @staticmethod
    def backward(ctx, d_raw):
        run, ctx.run = ctx.run, None
        if d_raw is None:  # the network's output did not reach the loss
            return (None, None, None) + (None,) * len(ctx.needs_input_grad[3:])
        if run is None:
            raise RuntimeError("backward through a network query a second time: its rows were released by the first")
        return (None, None, None) + tuple(run.gradients(nv.f32(d_raw).reshape(-1, 4)))
