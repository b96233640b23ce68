"""The reference's network (run_nerf_helpers.py:80-117) evaluated and trained layer by layer on the 8-bit
dense-layer kernels, for the widths and depths the fused kernels are not built for.

Every layer's input is held in 8-bit integers with one scale per point; a hidden layer is one launch that
reads the integers of the layer before and leaves its own (ops.linear_int8_quantized), so a point's
activations never exist in more than 8 bits, and the integers, scales and ReLU bits are all that the
backward pass keeps: about 2.8 KB per point of the 8 x 256 network, where the fused kernels save 4.7 KB.
Gradients between layers are bf16, parameter gradients fp32; rounding to 8 bits passes gradients on
unchanged.

    model = init_nerf_model(D=4, W=128, input_ch=63, input_ch_views=27, skips=[2], use_viewdirs=True,
                            precision='int8')
    render_kwargs_train, ... = create_nerf(args)        # args.precision = 'int8'
"""
import torch

from . import _native as nv
from . import ops
from .run_nerf_helpers import LaidOut, NerfModel

_QUERY_POINTS = 1 << 20   # points evaluated at a time when nothing is recorded: bounds the transient memory


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


def _encode(x, channels):
    return ops.embed(x, (channels - 3) // 6) if channels > 3 else x


class _Pass:
    """One forward pass: rows of every layer's input, in the order of split()."""

    def __init__(self, model, pts, viewdirs, S):
        """pts [P, 3], viewdirs [P / S, 3], all fp32."""
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
            # the narrow part of a concatenated input first, as the addend of the other
            self.inputs[i] = parts
            add = None
            at = [j for j, (_, _, enc) in enumerate(model.split(i)) if not enc or len(parts) == 1][0]
            for j, rows in enumerate(parts):
                if j != at:
                    add = ops.linear_int8(rows, packed[i][j], dtype=torch.bfloat16)
            if 'dtype' in out:
                return ops.linear_int8(parts[at], packed[i][at], model.bias(i), addend=add, **out)
            return ops.linear_int8_quantized(parts[at], packed[i][at], model.bias(i), addend=add, pow2=True, **out)

        h = [pe]
        for i in range(D):
            y = dense(i, h, relu=True, want_mask=True)
            h = [pe, y] if i in model.skips else [y]
        alpha = dense(D + 3, h, dtype=torch.float32)
        bott = dense(D, h)
        v = dense(D + 1, [bott, ve], relu=True, want_mask=True)
        rgb = dense(D + 2, [v], dtype=torch.float32)
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
    step = max(_QUERY_POINTS // S, 1)
    with torch.no_grad():
        out = [_Pass(model, pts[i * S:(i + step) * S], viewdirs[i:i + step], S).raw for i in range(0, P // S, step)]
    return out[0] if len(out) == 1 else torch.cat(out, 0)


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
