"""Attention with one decay per head against its recurrence in 64 bits.

Bounds are elementwise, in units of the sum of the magnitudes of the terms that make up a value: the same recurrence (or its
gradient, for gradients) on the magnitudes of the inputs.  A rounding to bf16 is off by at most 2^-8 of what is rounded.
  bf16 forward   scores or the state as an operand, the decayed values inside the state, and the result: three roundings.
  bf16 backward  operands in two planes (2^-16 each, twice in a row at most), and the result: one rounding.
  float32        three planes lose 2^-24; the tensor cores cut off up to 2^-23 of each of 16 + 1 additions of a 16-long sum, and
                 float32 additions of 16 such sums and of 12 chunks follow: below 64 x 2^-24.
The gradient of the gates is a sum from a token to the end of q dq - k dk, formed before these are rounded, so its unit is
that sum of magnitudes; the forward's final state enters with its own error.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F4, ALL_FINE = 2.0 ** -8, 64 * 2.0 ** -24, 2.0 ** -15


def recurrence(h, g, v, k, q):
    """h (B,H,Dk,Dv), g (B,T,H), v (B,T,H,Dv), k and q (B,T,Hk,Dk) in 64 bits."""
    rep = v.shape[2] // k.shape[2]
    k, q = k.repeat_interleave(rep, 2), q.repeat_interleave(rep, 2)
    outs = []
    for t in range(v.shape[1]):
        h = g[:, t].exp()[..., None, None] * h + k[:, t, :, :, None] * v[:, t, :, None, :]
        outs.append((q[:, t, :, :, None] * h).sum(-2))
    return h, torch.stack(outs, 1)


def make(dev, B, T, H, Hk, Dk, Dv, dtype, hdtype, seed=0, shift=2.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    g = torch.nn.functional.logsigmoid(n(B, T, H) + shift)
    return [n(B, H, Dk, Dv).to(hdtype), g, n(B, T, H, Dv).to(dtype), (n(B, T, Hk, Dk) * Dk ** -0.5).to(dtype), n(B, T, Hk, Dk).to(dtype)]


def with_grads(fn, xs, cots):
    xs = [x.detach().clone().requires_grad_(True) for x in xs]
    hf, out = fn(*xs)
    return [hf, out], list(torch.autograd.grad([hf, out], xs, cots))


def check(xs, cots, got, grads, dtype, hdtype, ctx=""):
    up = [x.double() for x in xs]
    (hf, out), want = with_grads(recurrence, up, [c.double() for c in cots])
    mags = [up[0].abs(), up[1], *(x.abs() for x in up[2:])]
    (mh, mo), mag = with_grads(recurrence, mags, [c.double().abs() for c in cots])
    ref, unit = [hf, out, *want], [mh, mo, *mag]
    rep = xs[2].shape[2] // xs[3].shape[2]
    # what the running sum of the gates' gradient adds up
    per_head = lambda x, d: (x * d).sum(-1).repeat_interleave(rep, 2) if x.shape[2] != xs[2].shape[2] else (x * d).sum(-1)  # noqa: E731
    run = (per_head(mags[4], mag[4]) + per_head(mags[3], mag[3])).flip(1).cumsum(1).flip(1)
    end = (mh * cots[0].double().abs()).sum((-1, -2))[:, None]
    f32 = dtype == torch.float32
    state = F4 if hdtype == torch.float32 else 2 * BF       # of the final state
    c = [state, F4 if f32 else 3 * BF]
    back = F4 if f32 else BF + ALL_FINE
    c += [F4 + (0 if f32 else ALL_FINE) if hdtype == torch.float32 else BF + ALL_FINE, None, back, back, back]
    for i, (a, b) in enumerate(zip([*got, *grads], ref)):
        name = ("hidden_final", "out", "dh", "dg", "dv", "dk", "dq")[i]
        if i == 3:
            lim = (F4 if f32 else ALL_FINE + F4) * (run + end) + (F4 if f32 or hdtype == torch.float32 else BF) * end
        else:
            lim = c[i] * unit[i]
        worst = ((a.double() - b).abs() - lim).max().item()
        assert torch.isfinite(a).all() and worst <= 1e-12, (ctx, name, worst, lim.max().item())


SIZES = [  # B, T, H, Hk, Dk, Dv
    (1, 1, 1, 1, 64, 64), (2, 2, 3, 1, 8, 8), (1, 63, 2, 2, 128, 128), (2, 64, 4, 2, 128, 64), (1, 65, 2, 1, 80, 96),
    (1, 130, 6, 2, 32, 136), (1, 200, 1, 1, 256, 256), (1, 777, 2, 1, 64, 128), (3, 96, 2, 2, 256, 40), (1, 1025, 1, 1, 128, 128),
]


@pytest.mark.parametrize("dtype,hdtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("size", SIZES)
def test_against_the_recurrence(cuda_device, size, dtype, hdtype):
    from gla_jax_b200 import chunk_decay_attention
    xs = make(cuda_device, *size, dtype, hdtype, seed=sum(size))
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    cots = [torch.randn(x.shape, generator=gen, device=cuda_device).to(x.dtype) for x in (xs[0], xs[2])]
    got, grads = with_grads(chunk_decay_attention, xs, cots)
    check(xs, cots, got, grads, dtype, hdtype, size)
    with torch.no_grad():
        hf, out = chunk_decay_attention(*xs)
    assert torch.equal(hf, got[0]) and torch.equal(out, got[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_differences_of_a_sharp_and_a_soft_gate(cuda_device, dtype):
    """The gates' gradient against central differences of the recurrence in 64 bits."""
    from gla_jax_b200 import chunk_decay_attention
    xs = make(cuda_device, 1, 70, 1, 1, 16, 16, dtype, torch.float32, seed=3, shift=0.0)
    cots = [torch.zeros_like(xs[0]), torch.randn_like(xs[2])]
    _, grads = with_grads(chunk_decay_attention, xs, cots)
    up, e = [x.double() for x in xs], 1e-4
    for t in (0, 1, 33, 64, 69):
        f = []
        for s in (e, -e):
            g = up[1].clone()
            g[0, t, 0] += s
            f.append((recurrence(up[0], g, *up[2:])[1] * cots[1].double()).sum())
        want = float(f[0] - f[1]) / (2 * e)
        # the difference itself: e^2 / 6 of the third derivative, which is that of a sum of exponentials; 1e-3 covers the rest
        assert abs(float(grads[1][0, t, 0]) - want) <= 1e-3 * max(1.0, abs(want)), t


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decays_of_the_head(cuda_device, dtype):
    """(H,) equals the same decay at every token; its gradient is the sum."""
    from gla_jax_b200 import chunk_decay_attention
    B, T, H = 2, 150, 4
    xs = make(cuda_device, B, T, H, 2, 64, 64, dtype, dtype)
    xs[1] = torch.tensor([-0.5, -0.01, 0.0, -3.0], device=cuda_device)
    cots = [torch.randn_like(xs[0]), torch.randn_like(xs[2])]
    wide = [xs[0], xs[1].expand(B, T, H).contiguous(), *xs[2:]]
    got, grads = with_grads(chunk_decay_attention, xs, cots)
    want, gw = with_grads(chunk_decay_attention, wide, cots)
    for a, b in zip([*got, *(grads[i] for i in (0, 2, 3, 4))], [*want, *(gw[i] for i in (0, 2, 3, 4))]):
        assert torch.equal(a, b)
    assert grads[1].shape == (H,)
    torch.testing.assert_close(grads[1], gw[1].sum((0, 1)), rtol=1e-4, atol=1e-3)
    with torch.no_grad():
        assert torch.equal(chunk_decay_attention(*xs)[1], got[1])


def test_one_sequence_views_and_gate_types(cuda_device):
    from gla_jax_b200 import chunk_decay_attention
    xs = make(cuda_device, 1, 90, 2, 2, 64, 64, torch.bfloat16, torch.float32)
    want = chunk_decay_attention(*xs)
    one = chunk_decay_attention(*(x[0] for x in xs))
    assert torch.equal(one[0], want[0][0]) and torch.equal(one[1], want[1][0])
    # views of a joint projection, and of rows that start anywhere
    joint = torch.cat([xs[2], xs[3], xs[4]], -1)
    got = chunk_decay_attention(xs[0], xs[1], *joint.split(64, -1))
    assert torch.equal(got[1], want[1])
    big = torch.zeros(1, 91, 2, 64, device=cuda_device, dtype=torch.bfloat16)
    big[:, 1:] = xs[4]
    assert torch.equal(chunk_decay_attention(*xs[:4], big[:, 1:])[1], want[1])
    g16 = xs[1].bfloat16()
    assert torch.equal(chunk_decay_attention(xs[0], g16, *xs[2:])[1], chunk_decay_attention(xs[0], g16.float(), *xs[2:])[1])
    leaf = g16.clone().requires_grad_(True)
    chunk_decay_attention(xs[0], leaf, *xs[2:])[1].float().sum().backward()
    assert leaf.grad.dtype == torch.bfloat16
    h, o = chunk_decay_attention(xs[0], xs[1][:, :0], *(x[:, :0] for x in xs[2:]))
    assert torch.equal(h, xs[0]) and o.shape == (1, 0, 2, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_resets_and_values_that_are_not_finite(cuda_device, dtype):
    from gla_jax_b200 import chunk_decay_attention
    xs = make(cuda_device, 1, 140, 2, 1, 64, 64, dtype, torch.float32, shift=5.0)
    h, g, v, k, q = xs
    g[0, 40, 0] = -math.inf
    g[0, 41, 0] = -1e30
    g[0, 77, 1] = -500.0
    hf, out = chunk_decay_attention(h, g, v, k, q)
    # what came before a reset is gone, so that the sequence from there on stands alone
    h2, o2 = chunk_decay_attention(torch.zeros_like(h), g[:, 41:].clone(), v[:, 41:], k[:, 41:], q[:, 41:])
    up = [x.double() for x in (h, g.clamp(min=-1e4), v, k, q)]
    rh, ro = recurrence(*up)
    mh, mo = recurrence(up[0].abs(), up[1], *(x.abs() for x in up[2:]))
    c = F4 if dtype == torch.float32 else 3 * BF
    assert ((out.double() - ro).abs() <= c * mo).all() and ((hf.double() - rh).abs() <= F4 * mh).all()
    assert ((h2 - hf)[0, 0].abs() <= 2 * F4 * mh[0, 0]).all()
    # values at token t that are not finite reach t and later only, keys and queries likewise
    for t, what in ((37, 2), (64, 2), (100, 3), (70, 4)):
        for bad in (math.nan, math.inf):
            ys = [x.clone() for x in xs]
            ys[what][0, t, 0, 5] = bad
            _, o = chunk_decay_attention(*ys)
            rest = [c for c in range(64) if c != 5 or what != 2]
            assert torch.equal(o[:, :t, :, rest], out[:, :t, :, rest]), (t, what, bad)
            # the value's own column: the same terms summed in another order, each sum within F4 of them, and in bf16
            # a rounding that may fall the other way
            near = 2 * F4 * mo[:, :t] + (BF * out[:, :t].double().abs() * 2 if dtype == torch.bfloat16 else 0)
            assert ((o[:, :t].double() - out[:, :t].double()).abs() <= near).all(), (t, what, bad)
            assert not torch.isfinite(o[0, t, 0]).all()
            if what == 2:
                clean = [c for c in range(64) if c != 5]
                assert torch.equal(o[0, :, :, clean], out[0, :, :, clean])
            if what == 4:
                assert torch.equal(o[:, t + 1:], out[:, t + 1:])


def _pack(dev, lens, H, Hk, Dk, Dv, dtype, seed=0):
    xs = make(dev, 1, sum(lens), H, Hk, Dk, Dv, dtype, dtype, seed)
    h = torch.randn(len(lens), H, Dk, Dv, device=dev).to(dtype)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return [h, *(x[0] for x in xs[1:])], cu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens", [[5], [1, 1, 1], [0, 64, 0, 0, 65, 1, 0], [300, 0, 513, 2], [700, 256, 256, 90, 0]])
def test_packed_equals_each_sequence(cuda_device, lens, dtype):
    from gla_jax_b200 import chunk_decay_attention, chunk_decay_attention_packed
    xs, cu = _pack(cuda_device, lens, 2, 1, 64, 96, dtype)
    cots = [torch.randn_like(xs[0]), torch.randn_like(xs[2])]
    dev_cu = torch.tensor(cu, dtype=torch.int32, device=cuda_device)
    got, grads = with_grads(lambda *a: chunk_decay_attention_packed(*a, dev_cu), xs, cots)
    tol = 2 * BF if dtype == torch.bfloat16 else 1e-4
    for s, (a, b) in enumerate(zip(cu, cu[1:])):
        one = [xs[0][s], *(x[a:b] for x in xs[1:])]
        if a == b:
            assert torch.equal(got[0][s], xs[0][s]) and torch.equal(grads[0][s], cots[0][s])
            continue
        w, gw = with_grads(chunk_decay_attention, one, [cots[0][s], cots[1][a:b]])
        pairs = [(got[0][s], w[0]), (got[1][a:b], w[1]), (grads[0][s], gw[0]), *((grads[i][a:b], gw[i]) for i in (1, 2, 3, 4))]
        for i, (x, y) in enumerate(pairs):
            # runs of a sequence are cut elsewhere, so that sums are rounded in another order
            assert (x.double() - y.double()).norm() <= tol * y.double().norm() + 1e-6, (s, i)
    listed, _ = with_grads(lambda *a: chunk_decay_attention_packed(*a, cu), xs, cots)
    assert torch.equal(listed[1], got[1]) and torch.equal(listed[0], got[0])


def test_packed_rows_behind_the_last_sequence_and_bad_offsets(cuda_device):
    from gla_jax_b200 import chunk_decay_attention_packed, check_device
    from gla_jax_b200._lib import GlaError
    check_device()
    xs, _ = _pack(cuda_device, [400, 300, 500], 2, 2, 64, 64, torch.bfloat16)
    xs[0] = xs[0][:2]
    cu = torch.tensor([0, 400, 700], dtype=torch.int32, device=cuda_device)
    cots = [torch.randn_like(xs[0]), torch.randn_like(xs[2])]
    got, grads = with_grads(lambda *a: chunk_decay_attention_packed(*a, cu), xs, cots)
    assert (got[1][700:] == 0).all() and all((grads[i][700:] == 0).all() for i in (1, 2, 3, 4))
    short = [xs[0], *(x[:700].clone() for x in xs[1:])]
    w, gw = with_grads(lambda *a: chunk_decay_attention_packed(*a, cu), short, [cots[0], cots[1][:700].clone()])
    assert (got[0].float() - w[0].float()).norm() <= 2 * BF * w[0].float().norm()
    assert (grads[2][:700].float() - gw[2].float()).norm() <= 2 * BF * gw[2].float().norm()
    check_device()
    for bad in ([0, 800, 700], [0, 5, 5000], [-3, 5, 9], [7, 9, 1200]):
        b = torch.tensor(bad, dtype=torch.int32, device=cuda_device)
        h, o = chunk_decay_attention_packed(*xs, b)
        with pytest.raises(GlaError):
            check_device()
    check_device()


def test_step_continues_a_prompt(cuda_device):
    """A prompt in one call, then tokens one by one, against the recurrence; state in float32."""
    from gla_jax_b200 import chunk_decay_attention, decay_attention_step
    for (B, T, H, Hk, Dk, Dv), dtype in (((2, 70, 4, 2, 128, 64), torch.bfloat16), ((1, 5, 2, 2, 8, 200), torch.float32), ((3, 33, 2, 1, 256, 256), torch.bfloat16)):
        xs = make(cuda_device, B, T + 3, H, Hk, Dk, Dv, dtype, torch.float32, seed=T)
        up = [x.double() for x in xs]
        _, ro = recurrence(*up)
        _, mo = recurrence(up[0].abs(), up[1], *(x.abs() for x in up[2:]))
        state, _ = chunk_decay_attention(xs[0], *(x[:, :T] for x in xs[1:]))
        c = F4 + (BF if dtype == torch.bfloat16 else 0)
        for t in range(T, T + 3):
            out = decay_attention_step(state, *(x[:, t] for x in xs[1:]))
            assert out.dtype == dtype and ((out.double() - ro[:, t]).abs() <= c * mo[:, t]).all()
        out = decay_attention_step(state, *(x[:, 0] for x in xs[1:]), out_dtype=torch.float32)
        assert out.dtype == torch.float32


def test_in_a_graph_and_on_another_stream(cuda_device):
    """Forward and backward captured and replayed with new inputs.  (No eager graph of the same leaves is alive: torch's
    engine then joins that graph's stream, which no capture survives, whatever the operator.)"""
    from gla_jax_b200 import chunk_decay_attention
    xs = make(cuda_device, 1, 600, 2, 1, 64, 64, torch.bfloat16, torch.bfloat16)
    leaves = [x.clone().requires_grad_(True) for x in xs]
    cots = [torch.randn_like(xs[0]), torch.randn_like(xs[2])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(chunk_decay_attention(*leaves), leaves, cots)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = chunk_decay_attention(*leaves)
        grads = torch.autograd.grad(outs, leaves, cots)
    new = make(cuda_device, 1, 600, 2, 1, 64, 64, torch.bfloat16, torch.bfloat16, seed=9)
    with torch.no_grad():
        for a, b in zip(leaves, new):
            a.copy_(b)
    graph.replay()
    want, gw = with_grads(chunk_decay_attention, new, cots)
    torch.cuda.synchronize()
    for a, b in zip([*outs, *grads], [*want, *gw]):
        assert torch.equal(a, b)


def test_refusals(cuda_device):
    from gla_jax_b200 import chunk_decay_attention as f, chunk_decay_attention_packed as fp, decay_attention_step as step
    h, g, v, k, q = make(cuda_device, 1, 16, 4, 2, 64, 64, torch.bfloat16, torch.float32)
    with pytest.raises(ValueError, match="multiple"):
        f(h, g, v, k[:, :, :1].expand(-1, -1, 3, -1), q[:, :, :1].expand(-1, -1, 3, -1))
    with pytest.raises(ValueError, match="hidden"):
        f(h[:, :2], g, v, k, q)
    with pytest.raises(ValueError, match="log_decay"):
        f(h, g[:, :5], v, k, q)
    with pytest.raises(ValueError, match="key and query"):
        f(h, g, v, k, q[:, :5])
    with pytest.raises(TypeError):
        f(h, g, v.half(), k.half(), q.half())
    with pytest.raises(TypeError):
        f(h, g, v, k.float(), q)
    with pytest.raises(RuntimeError, match="multiples of 8"):
        f(h[..., :60], g, v[..., :60], k, q)
    with pytest.raises(ValueError, match="CUDA|cuda|on "):
        f(h.cpu(), g, v, k, q)
    with pytest.raises(ValueError, match="rise"):
        fp(h.expand(2, -1, -1, -1), g[0], v[0], k[0], q[0], [0, 9, 8])
    with pytest.raises(ValueError, match="hidden_init"):
        fp(h, g[0], v[0], k[0], q[0], [0, 8, 16])
    state = h.clone()
    with pytest.raises(TypeError):
        step(state.bfloat16(), g[:, 0], v[:, 0], k[:, 0], q[:, 0])
    with pytest.raises(ValueError, match="parents"):
        step(state, g[:, 0], v[:, 0], k[:, 0], q[:, 0], parents=torch.zeros(2, 2, dtype=torch.int32, device=cuda_device))
    with pytest.raises(ValueError):
        step(state, g[:, 0], v[:, 0], k[:, 0, :, :8], q[:, 0])
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(NotImplementedError):
            f(h, g, fwd.make_dual(v, v), k, q)


@pytest.mark.parametrize("hdtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,Hk,Dk,Dv", [(4, 2, 128, 64), (2, 2, 64, 128), (1, 1, 128, 128), (2, 1, 40, 200)])
def test_gates_of_every_sharpness(cuda_device, H, Hk, Dk, Dv, hdtype):
    """Stretches of 128 tokens whose gates sum up to 2, 100, 200 and 800: weights of whole chunks, of groups, of pairs."""
    from gla_jax_b200 import chunk_decay_attention
    T = 5 * 128 + 37
    xs = make(cuda_device, 1, T, H, Hk, Dk, Dv, torch.bfloat16, hdtype, seed=Dk)
    rate = torch.tensor([0.015, 0.8, 1.6, 6.0, 0.3, 0.02], device=cuda_device)
    xs[1] = -rate.repeat_interleave(128)[:T, None] * (0.5 + torch.rand(1, T, H, device=cuda_device))
    cots = [torch.randn_like(xs[0]), torch.randn_like(xs[2])]
    got, grads = with_grads(chunk_decay_attention, xs, cots)
    check(xs, cots, got, grads, torch.bfloat16, hdtype, (Dk, Dv))


@pytest.mark.parametrize("shift", [5.0, -3.0])
@pytest.mark.parametrize("D", [64, 128])
def test_gradients_that_are_not_finite_stay_with_earlier_tokens(cuda_device, D, shift):
    """A cotangent or a query that is not finite at token t reaches the gradients of tokens up to t of its own head."""
    from gla_jax_b200 import chunk_decay_attention
    xs = make(cuda_device, 1, 300, 2, 2, D, D, torch.bfloat16, torch.float32, shift=shift)
    cots = [torch.randn_like(xs[0]), torch.randn_like(xs[2])]
    _, want = with_grads(chunk_decay_attention, xs, cots)
    mags = [xs[0].double().abs(), xs[1].double(), *(x.double().abs() for x in xs[2:])]
    _, mag = with_grads(recurrence, mags, [c.double().abs() for c in cots])
    for t in (37, 127, 128, 201):
        for bad in (math.nan, math.inf):
            for what in ("cotangent", "query"):
                ys, cs = [x.clone() for x in xs], [c.clone() for c in cots]
                (cs[1] if what == "cotangent" else ys[4])[0, t, 0, 5] = bad
                _, got = with_grads(chunk_decay_attention, ys, cs)
                for i in (1, 2, 3, 4):
                    assert torch.equal(got[i][:, :, 1], want[i][:, :, 1]), (t, bad, what, i)
                for i in (2, 3, 4):
                    # terms summed in another order, each sum within F4 of them, and a rounding that may fall the other way
                    a, b = got[i][:, t + 1:, 0].double(), want[i][:, t + 1:, 0].double()
                    assert ((a - b).abs() <= 2 * F4 * mag[i][:, t + 1:, 0] + 2 * BF * b.abs()).all(), (t, bad, what, i)
                assert torch.isfinite(got[1][:, t + 1:]).all()
                if what == "query":
                    assert torch.equal(got[4][:, :t], want[4][:, :t])            # (its own gradient does not read it)
                    assert not torch.isfinite(got[3][0, t, 0]).all()
                else:
                    assert not torch.isfinite(got[2][0, t, 0]).all()


def test_two_streams_at_once(cuda_device):
    from gla_jax_b200 import chunk_decay_attention
    xs = [make(cuda_device, 2, 1500, 3, 3, 128, 128, torch.bfloat16, torch.bfloat16, seed=s) for s in (1, 2)]
    cots = [torch.randn_like(xs[0][0]), torch.randn_like(xs[0][2])]
    want = [with_grads(chunk_decay_attention, x, cots) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for i in (0, 1):
            streams[i].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[i]):
                got[i] = with_grads(chunk_decay_attention, xs[i], cots)
    torch.cuda.synchronize()
    for (a, ga), (b, gb) in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip([*a, *ga], [*b, *gb]))


@pytest.mark.parametrize("rate", [0.02, 0.45, 2.0])
def test_large_scores_under_decay(cuda_device, rate):
    """Queries and keys of 2^14 each, so that scores reach 2^35: nothing between the inputs and the results may overflow."""
    from gla_jax_b200 import chunk_decay_attention
    xs = make(cuda_device, 1, 260, 2, 2, 128, 128, torch.bfloat16, torch.float32)
    xs[1] = torch.full_like(xs[1], -rate)
    xs[3], xs[4] = xs[3] * 2.0 ** 17, xs[4] * 2.0 ** 14
    cots = [torch.randn_like(xs[0]), torch.randn_like(xs[2])]
    got, grads = with_grads(chunk_decay_attention, xs, cots)
    check(xs, cots, got, grads, torch.bfloat16, torch.float32, rate)


def test_gradients_of_a_part_of_the_results(cuda_device):
    """Either result alone, and any subset of the arguments, against all of them."""
    from gla_jax_b200 import chunk_decay_attention
    for dtype in (torch.bfloat16, torch.float32):
        xs = make(cuda_device, 2, 150, 4, 2, 64, 64, dtype, dtype)
        cots = [torch.randn_like(xs[0]), torch.randn_like(xs[2])]
        zero = [torch.zeros_like(c) for c in cots]
        for keep in (0, 1):
            _, want = with_grads(chunk_decay_attention, xs, [c if i == keep else zero[i] for i, c in enumerate(cots)])
            leaves = [x.clone().requires_grad_(True) for x in xs]
            got = torch.autograd.grad(chunk_decay_attention(*leaves)[keep], leaves, cots[keep])
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        _, want = with_grads(chunk_decay_attention, xs, cots)
        for which in ((0,), (1,), (2,), (3,), (4,), (1, 4), (0, 2, 3)):
            leaves = [x.clone().requires_grad_(i in which) for i, x in enumerate(xs)]
            got = torch.autograd.grad(chunk_decay_attention(*leaves), [leaves[i] for i in which], cots)
            # (without the gates' gradient the others need one plane of the state less)
            for i, a in zip(which, got):
                assert (a.double() - want[i].double()).norm() <= (2 * BF if dtype == torch.bfloat16 else 1e-5) * want[i].double().norm(), (which, i)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_arrays_that_start_anywhere(cuda_device, dtype):
    """Contiguous arrays off 16 bytes, as slices of a flat buffer are, cotangents among them."""
    from gla_jax_b200 import chunk_decay_attention, decay_attention_step

    def moved(x):
        flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:]
        return flat.copy_(x.flatten()).view(x.shape)

    xs = make(cuda_device, 1, 300, 2, 1, 64, 64, dtype, dtype)
    cots = [torch.randn_like(xs[0]), torch.randn_like(xs[2])]
    got, want = [], []
    for res, f in ((want, lambda x: x), (got, moved)):
        leaves = [f(x).requires_grad_(True) for x in xs]
        outs = chunk_decay_attention(*leaves)
        res += [*outs, *torch.autograd.grad(outs, leaves, [f(c) for c in cots])]
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), i
    state = xs[0].float()
    a, b = state.clone(), state.clone()
    o1 = decay_attention_step(a, xs[1][:, 0], *(x[:, 0] for x in xs[2:]))
    o2 = decay_attention_step(b, moved(xs[1][:, 0].contiguous()), *(moved(x[:, 0].contiguous()) for x in xs[2:]))
    assert torch.equal(a, b) and torch.equal(o1, o2)
