"""The fused join of residual, gate and norms against 64 bits.

Tolerances.  A stored value is off by half a step of its type.  Before that, everything is fp32: a
row's sums run over at most 16 values a thread, five shuffles and 16 warps, so with H = 2^-24 a
mean or mean square is off by less than 40 H of its terms' magnitudes, and a value that takes two
such sums, a root and some ten products by less than 64 H of the magnitudes it is made of (two
chained norms: 256 H).  Parameter gradients add rows one after another in fp32: their bound grows
with the rows that a block and the final sum add up (ROWS / 592 + 592 / 16 + 32 with their terms'
own 256, under 512 for the sizes here).  The norm that follows and the backward pass are held to
the stream that the kernel returned."""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
H = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _floor(dtype):
    return 2.0 ** -25 if dtype is F16 else 0.0            # half the smallest step of fp16


def _close(got, want, magnitude, rel, what):
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    limit = _half(got.dtype) * want.abs() * 1.001 + rel * magnitude + _floor(got.dtype) + 1e-37
    worst = ((got.double() - want).abs() / limit).max() if got.numel() else torch.zeros(())
    assert worst <= 1, (what, float(worst))


class Case:
    """Inputs, the kernel's results, and what 64 bits say."""

    def __init__(self, shape, kind="rms", stream=BF16, low=BF16, params=F32, post=True, gate="channel",
                 next=True, biases=None, scale=0.5, seed=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        d = shape[-1]
        biases = kind == "layer" if biases is None else biases

        def normal(*s, dtype=F32, std=1.0, mean=0.0):
            return (torch.randn(*s, device=DEV, generator=g) * std + mean).to(dtype).requires_grad_(True)

        self.kind, self.scale, self.low, self.d = kind, scale, low, d
        self.residual, self.update = normal(*shape, dtype=stream, std=1.5, mean=0.3), normal(*shape, dtype=low, std=0.6, mean=-0.1)
        self.weight = normal(d, dtype=params, std=0.2, mean=1.0) if next else None
        self.bias = normal(d, dtype=params, std=0.1) if next and biases else None
        self.post_weight = normal(d, dtype=params, std=0.2, mean=1.0) if post else None
        self.post_bias = normal(d, dtype=params, std=0.1) if post and biases else None
        self.gate = None
        if gate == "channel":
            self.gate = normal(d, dtype=params, std=0.3, mean=0.8)
        elif gate == "sequence":
            self.gate = normal(shape[0], *(1,) * (len(shape) - 2), d, dtype=params, std=0.3, mean=0.8)
        self.d_stream = torch.randn(*shape, device=DEV, generator=g).to(stream)
        self.d_normed = torch.randn(*shape, device=DEV, generator=g).to(low) if next else None

    def names(self):
        return [n for n in ("residual", "update", "weight", "bias", "post_weight", "post_bias", "gate")
                if getattr(self, n) is not None]

    def run(self, d_stream="given", d_normed="given"):
        from gpubridge_b200.ops.residual_norm import residual_norm
        self.stream, self.normed = residual_norm(
            self.residual, self.update, self.weight, self.bias, post_weight=self.post_weight,
            post_bias=self.post_bias, gate=self.gate, scale=self.scale, kind=self.kind, out_dtype=self.low)
        pairs = [(self.stream, self.d_stream if d_stream == "given" else d_stream),
                 (self.normed, self.d_normed if d_normed == "given" else d_normed)]
        pairs = [(o, g) for o, g in pairs if o is not None and g is not None]
        grads = torch.autograd.grad([o for o, _ in pairs], [getattr(self, n) for n in self.names()],
                                    [g for _, g in pairs], allow_unused=True)
        self.grads = dict(zip(self.names(), grads))
        self.used = ([g for o, g in pairs if o is self.stream] or [None])[0], \
                    ([g for o, g in pairs if o is self.normed and o is not None] or [None])[0]
        return self

    def check(self):
        w = lambda t: None if t is None else t.detach().double()  # noqa: E731
        layer, s, d = self.kind == "layer", self.scale, self.d
        r, u, ds, dy = w(self.residual), w(self.update), *map(w, self.used)
        gate = w(self.gate) if self.gate is not None else torch.ones(d, dtype=torch.float64, device=DEV)

        def stats(x):
            mean = x.mean(-1, keepdim=True) if layer else torch.zeros_like(x[..., :1])
            rstd = ((x - mean).square().mean(-1, keepdim=True) + 1e-5).rsqrt()
            return (x - mean) * rstd, (x.abs() + (x.abs().mean(-1, keepdim=True) if layer else 0)) * rstd, rstd

        def back(g, size, hat, hat_size, rstd):
            """norm' of g, and of its magnitude"""
            got = g - hat * (g * hat).mean(-1, keepdim=True)
            big = size + hat_size * (size * hat_size).mean(-1, keepdim=True)
            if layer:
                got, big = got - g.mean(-1, keepdim=True), big + size.mean(-1, keepdim=True)
            return rstd * got, rstd * big

        v, v_size = u, u.abs()
        if self.post_weight is not None:
            uhat, uhat_size, urstd = stats(u)
            pb = w(self.post_bias) if self.post_bias is not None else torch.zeros(d, dtype=torch.float64, device=DEV)
            v, v_size = uhat * w(self.post_weight) + pb, uhat_size * w(self.post_weight).abs() + pb.abs()
        _close(self.stream, r + s * gate * v, r.abs() + abs(s) * gate.abs() * v_size, 64 * H, "stream")
        x = w(self.stream)
        hat, hat_size, rstd = stats(x)
        if self.normed is not None:
            b = w(self.bias) if self.bias is not None else torch.zeros(d, dtype=torch.float64, device=DEV)
            _close(self.normed, hat * w(self.weight) + b, hat_size * w(self.weight).abs() + b.abs(), 64 * H, "normed")
        dr = torch.zeros_like(x) if ds is None else ds
        dr_size = dr.abs()
        flat = lambda t: t.reshape(-1, d).sum(0)  # noqa: E731
        if dy is not None:
            got, big = back(dy * w(self.weight), dy.abs() * w(self.weight).abs(), hat, hat_size, rstd)
            dr, dr_size = dr + got, dr_size + big
            _close(self.grads["weight"], flat(dy * hat), flat(dy.abs() * hat_size), 512 * H, "d_weight")
            if self.bias is not None:
                _close(self.grads["bias"], flat(dy), flat(dy.abs()), 512 * H, "d_bias")
        elif self.weight is not None:
            assert self.grads["weight"] is None
        _close(self.grads["residual"], dr, dr_size, 128 * H, "d_residual")
        dv, dv_size = s * dr, abs(s) * dr_size
        if self.gate is not None:
            if self.gate.dim() == 1:
                add = flat
            else:
                add = lambda t: t.reshape(t.shape[0], -1, d).sum(1).view(self.gate.shape)  # noqa: E731
            _close(self.grads["gate"], add(dv * v), add(dv_size * v_size), 512 * H, "d_gate")
            dv, dv_size = dv * gate, dv_size * gate.abs()
        if self.post_weight is not None:
            _close(self.grads["post_weight"], flat(dv * uhat), flat(dv_size * uhat_size), 512 * H, "d_post_weight")
            if self.post_bias is not None:
                _close(self.grads["post_bias"], flat(dv), flat(dv_size), 512 * H, "d_post_bias")
            pw = w(self.post_weight)
            dv, dv_size = back(dv * pw, dv_size * pw.abs(), uhat, uhat_size, urstd)
        _close(self.grads["update"], dv, dv_size, 256 * H, "d_update")


TYPES = {"fp32": (F32, F32, F32), "autocast": (F32, BF16, F32), "autocast-fp16": (F32, F16, F32),
         "bf16": (BF16, BF16, BF16), "bf16-fp32-params": (BF16, BF16, F32), "fp16": (F16, F16, F16)}


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("width", [8, 100, 768, 1001, 1500, 2047, 2048])
def test_types_and_widths(types, kind, width):
    stream, low, params = TYPES[types]
    Case((3, 37, width), kind, stream, low, params, gate="sequence", seed=width).run().check()


@pytest.mark.parametrize("width", [1, 2, 3, 7, 31, 33, 256, 264, 511, 4096, 4097, 4104, 5000, 8191, 8192])
def test_every_kind_of_width(width):
    Case((2, 9, width), "layer", F32, F32, F32, gate="sequence", seed=width).run().check()
    Case((2, 9, width), "rms", BF16, BF16, BF16, seed=width).run().check()


@pytest.mark.parametrize("post,gate,next,biases", list(itertools.product(
    [False, True], ["none", "channel", "sequence"], [False, True], [False, True])))
def test_every_form(post, gate, next, biases):
    for kind, width in (("rms", 256), ("layer", 97)):
        Case((4, 5, width), kind, F32, BF16, F32, post, gate, next, biases, scale=-1.5).run().check()


@pytest.mark.parametrize("rows", [1, 2, 147, 148, 149, 593, 1185, 2400])
def test_row_counts(rows):
    Case((rows, 128), "rms", BF16, BF16, F32, gate="channel", seed=rows).run().check()
    Case((1, rows, 776), "layer", F32, BF16, F32, gate="sequence", seed=rows).run().check()


@pytest.mark.parametrize("batch,seq", [(1, 700), (7, 100), (100, 7), (700, 1), (2500, 1), (1300, 2), (13, 181)])
def test_gates_of_many_sequences(batch, seq):
    """Sequences longer than a block's share of the rows, shorter, and of one row."""
    Case((batch, seq, 64), "rms", F32, F32, F32, gate="sequence", seed=batch).run().check()


def test_four_dimensions_and_one():
    Case((2, 3, 5, 48), "rms", F32, F32, F32, gate="sequence").run().check()
    Case((40,), "layer", F32, F32, F32, gate="channel").run().check()
    Case((6, 40), "rms", F32, F32, F32, gate="sequence").run().check()


@pytest.mark.parametrize("which", ["stream", "normed"])
def test_only_one_output_is_used(which):
    case = Case((3, 17, 264), "layer", F32, BF16, F32, gate="sequence")
    (case.run(d_normed=None) if which == "stream" else case.run(d_stream=None)).check()


@pytest.mark.parametrize("view", ["inner", "transposed", "odd start", "every other", "dense"])
@pytest.mark.parametrize("low", [F32, BF16])
def test_strided_inputs_and_expanded_gradients(view, low):
    base = torch.randn(5, 12, 96, device=DEV).to(low).requires_grad_(True)
    residual = {"inner": base[:, 2:9, 16:80], "transposed": base.transpose(0, 1)[:, :, :64],
                "odd start": base[..., 1:65], "every other": base[:, ::2, :64], "dense": base}[view]
    case = Case(tuple(residual.shape), "rms", low, low, F32, gate="sequence")
    case.residual = residual
    update = case.update.detach().transpose(0, 1).contiguous().transpose(0, 1)
    case.update = update.requires_grad_(True)
    case.d_stream = torch.full((1, 1, 1), 0.5, device=DEV, dtype=low).expand(residual.shape)
    case.d_normed = torch.randn(residual.shape[-1], device=DEV).to(low).expand(residual.shape)
    case.run().check()


def test_no_rows():
    from gpubridge_b200.ops.residual_norm import residual_norm
    r, u = (torch.zeros(0, 4, 32, device=DEV, requires_grad=True) for _ in range(2))
    w = torch.ones(32, device=DEV, requires_grad=True)
    stream, normed = residual_norm(r, u, w, post_weight=w)
    assert stream.shape == normed.shape == (0, 4, 32)
    (stream.sum() + normed.sum()).backward()
    assert (w.grad == 0).all() and r.grad.shape == r.shape


def test_infinities_and_nan_stay_in_their_rows():
    from gpubridge_b200.ops.residual_norm import residual_norm
    r, u = torch.randn(9, 256, device=DEV), torch.randn(9, 256, device=DEV)
    w = torch.ones(256, device=DEV)
    clean = residual_norm(r, u, w, post_weight=w)
    r[2, 5], u[6, 0] = math.nan, math.inf
    got = residual_norm(r, u, w, post_weight=w)
    keep = [0, 1, 3, 4, 5, 7, 8]
    assert torch.equal(got.normed[keep], clean.normed[keep]) and torch.equal(got.stream[keep], clean.stream[keep])
    assert got.normed[2].isnan().all() and got.normed[6].isnan().any()


def test_large_offsets_and_zero_rows():
    """Rows of zeros have the norm's eps under the root; values far from zero keep their variance."""
    from gpubridge_b200.ops.residual_norm import residual_norm
    z = torch.zeros(3, 512, device=DEV)
    got = residual_norm(z, z, torch.ones(512, device=DEV), post_weight=torch.ones(512, device=DEV))
    assert (got.normed == 0).all()
    x = torch.randn(4, 512, device=DEV) + 1000.0
    got = residual_norm(x, z[:1].expand(4, 512), torch.ones(512, device=DEV), kind="layer").normed
    wide = x.double() - x.double().mean(-1, keepdim=True)
    want = wide / (wide.square().mean(-1, keepdim=True) + 1e-5).sqrt()
    # the mean of values near 1000 is off by up to 40 half steps of 1000
    assert (got.double() - want).abs().max() <= 2 * 40 * H * 1000


def test_autocast_gives_the_type_of_the_next_product():
    from gpubridge_b200.ops.residual_norm import residual_norm
    r, u = torch.randn(4, 64, device=DEV), torch.randn(4, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        stream, normed = residual_norm(r, u, w)
    assert stream.dtype == torch.float32 and normed.dtype == torch.bfloat16
    # nothing was rounded before the norm's result: stream and update in fp32 are joined in fp32
    assert torch.equal(stream, r + u)
    full = residual_norm(r, u, w)
    assert torch.equal(full.stream, stream) and torch.equal(full.normed.bfloat16(), normed)
    r.requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = residual_norm(r, u, w)
    grad, = torch.autograd.grad(out.normed.float().sum(), r)
    assert grad.dtype == torch.float32 and torch.isfinite(grad).all()


@pytest.mark.parametrize("scale", [1.0, 0.5])
@pytest.mark.parametrize("stream,low", [(BF16, BF16), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("width", [100, 512])
def test_plain_joins(scale, stream, low, width):
    """Without a post norm or a gate; with and without the following norm's gradient."""
    Case((3, 17, width), "rms", stream, low, F32, post=False, gate="none", scale=scale).run().check()
    Case((3, 17, width), "layer", stream, low, F32, post=False, gate="none", scale=scale).run(d_normed=None).check()
    Case((3, 17, width), "rms", stream, low, F32, post=False, gate="none", next=False, scale=scale).run().check()


def test_gradients_that_are_alike_do_not_share_memory():
    from gpubridge_b200.ops.residual_norm import residual_norm
    r, u = (torch.randn(4, 64, device=DEV, requires_grad=True) for _ in range(2))
    w = torch.ones(64, device=DEV)
    for weight in (w, None):
        r.grad = u.grad = None
        for _ in range(2):
            out = residual_norm(r, u, weight)
            (out.stream.square().sum() + (out.normed.sum() if weight is not None else 0)).backward()
        assert torch.equal(r.grad, u.grad) and r.grad.data_ptr() != u.grad.data_ptr()
        before = u.grad.clone()
        r.grad.zero_()
        assert torch.equal(u.grad, before)


def test_differences():
    """The gradients against differences of the plain form in 64 bits (CPU), and the kernel's
    gradients against those of the plain form."""
    from gpubridge_b200.ops.residual_norm import residual_norm
    g = torch.Generator().manual_seed(1)
    args = [torch.randn(2, 3, 5, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2)]
    params = [torch.randn(5, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(4)]
    gate = torch.randn(2, 1, 5, generator=g, dtype=torch.float64, requires_grad=True)
    for kind in ("rms", "layer"):
        def f(r, u, w, b, pw, pb, gate):
            return tuple(residual_norm(r, u, w, b, post_weight=pw, post_bias=pb, gate=gate, scale=0.3, kind=kind))
        assert torch.autograd.gradcheck(f, (*args, *params, gate))
        leaves = (*args, *params, gate)
        want = torch.autograd.grad([t.sum() + t.square().sum() for t in f(*leaves)], leaves)
        on = [t.detach().float().to(DEV).requires_grad_(True) for t in leaves]
        got = torch.autograd.grad([t.sum() + t.square().sum() for t in f(*on)], on)
        for a, b in zip(got, want):
            assert torch.allclose(a.double().cpu(), b, rtol=1e-4, atol=1e-4)


def test_same_bits_every_time():
    a = Case((4, 333, 768), "layer", F32, BF16, F32, gate="sequence").run()
    first = {k: v.clone() for k, v in a.grads.items()}
    a.run()
    assert all(torch.equal(a.grads[k], first[k]) for k in first)


def test_streams_and_a_replayed_training_step():
    from gpubridge_b200.ops.residual_norm import residual_norm
    case = Case((4, 100, 512), "rms", BF16, BF16, BF16, gate="sequence")
    eager = case.run()
    want = {k: v.clone() for k, v in eager.grads.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = Case((4, 100, 512), "rms", BF16, BF16, BF16, gate="sequence", seed=5)
    with torch.cuda.stream(side):
        other.run()
    case.run()
    torch.cuda.synchronize()
    other.check()
    assert all(torch.equal(case.grads[k], want[k]) for k in want)
    # captured with leaves of its own, replayed on new values
    leaves = [t.detach().clone().requires_grad_(True) for t in (case.residual, case.update, case.weight, case.gate)]
    graph = torch.cuda.CUDAGraph()
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())

    def step():
        s, n = residual_norm(leaves[0], leaves[1], leaves[2], gate=leaves[3])
        return s, n, torch.autograd.grad([s, n], leaves, [case.d_stream, case.d_normed])

    with torch.cuda.stream(warm):
        step()
    torch.cuda.current_stream().wait_stream(warm)
    with torch.cuda.graph(graph):
        s, n, grads = step()
    with torch.no_grad():
        leaves[0].copy_(other.residual)
        leaves[1].copy_(other.update)
    graph.replay()
    torch.cuda.synchronize()
    s2, n2, grads2 = step()
    assert torch.equal(s, s2) and torch.equal(n, n2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))


def test_refusals_on_the_gpu():
    from gpubridge_b200.ops.residual_norm import residual_norm
    x = torch.randn(2, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    with pytest.raises(ValueError, match="8192"):
        residual_norm(torch.zeros(1, 8193, device=DEV), torch.zeros(1, 8193, device=DEV))
    with pytest.raises(ValueError, match="float32, bfloat16"):
        residual_norm(x.double(), x.double())
    with pytest.raises(ValueError, match="same type"):
        residual_norm(x.bfloat16(), x.bfloat16(), w, out_dtype=torch.float32)
    with pytest.raises(ValueError, match="weight is on cpu"):
        residual_norm(x, x, w.cpu())
    stream, normed = residual_norm(x.requires_grad_(True), x, w)
    (g,) = torch.autograd.grad(normed.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
