"""Decay attention at the edges of what its documentation allows: offsets that fall, inputs that are not finite, many sequences."""
import math

import pytest
import torch

from test_gpu_decay import ALL_FINE, BF, F4, check, make, recurrence, with_grads

pytestmark = pytest.mark.gpu


def packed(dev, nseq, T, H, Hk, Dk, Dv, dtype, seed=0):
    xs = make(dev, 1, T, H, Hk, Dk, Dv, dtype, dtype, seed)
    gen = torch.Generator(device=dev).manual_seed(seed + 1)
    n = lambda *s: torch.randn(*s, generator=gen, device=dev).to(dtype)  # noqa: E731
    xs = [n(nseq, H, Dk, Dv), *(x[0] for x in xs[1:])]
    return xs, [n(nseq, H, Dk, Dv), n(T, H, Dv)]


def held_inside(offsets, T):
    """What offsets are taken as: rising from 0, none beyond T."""
    out = [0]
    for x in offsets[1:]:
        out.append(max(out[-1], min(max(x, 0), T)))
    return out


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 136)])
@pytest.mark.parametrize("offsets", [[0, 1000, 10, 1200], [0, 600, 300, 1200], [0, 1100, 100, 300, 1200], [7, 9, 1200], [-3, 500, -1, 900],
                                     [0, 5000, 3, 1100], [900, 800, 700], [0, 0, 2 ** 31 - 1, -2 ** 31, 1200]])
def test_offsets_that_fall_or_leave_the_axis(cuda_device, offsets, dtype, D):
    """1200 tokens of 2 heads are cut into runs: every row, state and gradient is what rising offsets give, and the call is reported."""
    from gla_jax_b200 import check_device, chunk_decay_attention_packed
    from gla_jax_b200._lib import GlaError
    T, nseq = 1200, len(offsets) - 1
    xs, cots = packed(cuda_device, nseq, T, 2, 1, D, D, dtype)
    bad, good = (torch.tensor(c, dtype=torch.int32, device=cuda_device) for c in (offsets, held_inside(offsets, T)))
    check_device()
    want, gw = with_grads(lambda *a: chunk_decay_attention_packed(*a, good), xs, cots)
    check_device()
    got, gg = with_grads(lambda *a: chunk_decay_attention_packed(*a, bad), xs, cots)
    with pytest.raises(GlaError, match="sequence"):
        check_device()
    for i, (a, b) in enumerate(zip([*got, *gg], [*want, *gw])):
        assert torch.equal(a, b), i
    end = int(good[-1])
    assert (got[1][end:] == 0).all() and all((gg[i][end:] == 0).all() for i in (1, 2, 3, 4))
    with torch.no_grad():
        hf, out = chunk_decay_attention_packed(*xs, bad)
    assert torch.equal(hf, want[0]) and torch.equal(out, want[1])
    with pytest.raises(GlaError):
        check_device()


def test_offsets_of_many_sequences(cuda_device):
    """More offsets than a pass over them takes at once, one in three falling."""
    from gla_jax_b200 import check_device, chunk_decay_attention_packed
    from gla_jax_b200._lib import GlaError
    T, nseq = 3000, 700
    gen = torch.Generator().manual_seed(2)
    cu = torch.randint(0, T + 1, (nseq - 1,), generator=gen).sort().values.tolist()
    offsets = [0, *(x - 40 * (i % 3 == 0) for i, x in enumerate(cu)), T]
    xs, cots = packed(cuda_device, nseq, T, 1, 1, 32, 32, torch.bfloat16)
    bad, good = (torch.tensor(c, dtype=torch.int32, device=cuda_device) for c in (offsets, held_inside(offsets, T)))
    want, gw = with_grads(lambda *a: chunk_decay_attention_packed(*a, good), xs, cots)
    check_device()
    got, gg = with_grads(lambda *a: chunk_decay_attention_packed(*a, bad), xs, cots)
    with pytest.raises(GlaError):
        check_device()
    assert all(torch.equal(a, b) for a, b in zip([*got, *gg], [*want, *gw]))


@pytest.mark.parametrize("dtype,hdtype,D", [(torch.bfloat16, torch.float32, 64), (torch.bfloat16, torch.bfloat16, 128), (torch.bfloat16, torch.bfloat16, 136),
                                            (torch.float32, torch.float32, 64)])
@pytest.mark.parametrize("T", [300, 900])
def test_gates_gradient_before_a_value_or_key_that_is_not_finite(cuda_device, T, dtype, hdtype, D):
    """dg_s = <exp(g_s) S_{s-1}, dS_s> reads values and keys before s only.  900 tokens of 2 heads are cut into runs.

    The gradient may be summed from either end, so the unit is everything that either sum adds up: the terms of all tokens, and
    the products of states and their gradients at both ends (which the states' own type rounds).  That bound is for errors which all
    fall the same way; as they fall, a rounded state's inner product is off by 2^-9 of its own size or so: 2^-7 of the largest."""
    from gla_jax_b200 import chunk_decay_attention
    xs = make(cuda_device, 1, T, 2, 1, D, D, dtype, hdtype, shift=4.0)
    gen = torch.Generator(device=cuda_device).manual_seed(4)
    cots = [torch.randn(x.shape, generator=gen, device=cuda_device).to(x.dtype) for x in (xs[0], xs[2])]
    _, want = with_grads(recurrence, [x.double() for x in xs], [c.double() for c in cots])
    mags = [xs[0].double().abs(), xs[1].double(), *(x.double().abs() for x in xs[2:])]
    (mh, _), mag = with_grads(recurrence, mags, [c.double().abs() for c in cots])
    per_head = lambda x, d: (x * d).sum(-1).repeat_interleave(2, 2)  # noqa: E731
    terms = (per_head(mags[4], mag[4]) + per_head(mags[3], mag[3])).sum(1)
    ends = (mh * cots[0].double().abs()).sum((-1, -2)) + (mags[0] * mag[0]).sum((-1, -2))
    fine = F4 if dtype == torch.float32 else ALL_FINE + F4
    lim = 2 * (fine * (terms + ends) + (F4 if hdtype == torch.float32 else BF) * ends)          # (1, H)
    for t in (0, 5, 130, T - 1):
        for what in (2, 3):
            for bad in (math.nan, math.inf):
                ys = [x.clone() for x in xs]
                ys[what][0, t, 0, 3] = bad
                _, got = with_grads(chunk_decay_attention, ys, cots)
                heads = 1 if what == 2 else 2                    # (the key is shared by both value heads)
                near = (got[1][:, : t + 1].double() - want[1][:, : t + 1]).abs()
                assert (near <= lim).all(), (t, what, bad, near.max().item(), lim.min().item())
                assert near.max() <= 2.0 ** -7 * want[1].abs().max(), (t, what, bad, near.max().item(), want[1].abs().max().item())
                assert not torch.isfinite(got[1][:, t + 1:, :heads]).any(), (t, what, bad)
                if what == 2:
                    assert ((got[1][:, :, 1].double() - want[1][:, :, 1]).abs() <= lim[:, 1]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_sequences_than_a_grid_is_high(cuda_device, dtype):
    """70,000 sequences of 0 to 3 tokens, as a batch and packed, equal the halves of them."""
    from gla_jax_b200 import chunk_decay_attention, chunk_decay_attention_packed
    n, half = 70000, 35000
    xs = make(cuda_device, n, 2, 1, 1, 8, 8, dtype, dtype)
    cots = [torch.randn_like(xs[0]), torch.randn_like(xs[2])]
    got, grads = with_grads(chunk_decay_attention, xs, cots)
    for s in (slice(0, half), slice(half, n)):
        want, gw = with_grads(chunk_decay_attention, [x[s] for x in xs], [c[s] for c in cots])
        assert all(torch.equal(a[s], b) for a, b in zip([*got, *grads], [*want, *gw]))
    cu = [0, *(torch.arange(n) % 4).cumsum(0).tolist()]
    xs, cots = packed(cuda_device, n, cu[-1], 1, 1, 8, 8, dtype)
    got, grads = with_grads(lambda *a: chunk_decay_attention_packed(*a, cu), xs, cots)
    for a, b in ((0, half), (half, n)):
        s, t = slice(a, b), slice(cu[a], cu[b])
        part = [x - cu[a] for x in cu[a:b + 1]]
        want, gw = with_grads(lambda *y: chunk_decay_attention_packed(*y, part), [xs[0][s], *(x[t] for x in xs[1:])], [cots[0][s], cots[1][t]])
        for i, (x, y) in enumerate(zip([*got, *grads], [*want, *gw])):
            assert torch.equal(x[s if i in (0, 2) else t], y), i


def test_bf16_decays_of_the_head_round_their_gradient_once(cuda_device):
    from gla_jax_b200 import chunk_decay_attention
    xs = make(cuda_device, 2, 500, 4, 4, 64, 64, torch.bfloat16, torch.bfloat16)
    cots = [torch.randn_like(xs[0]), torch.randn_like(xs[2])]
    xs[1] = torch.tensor([-0.5, -0.01, -0.1, -1.5], device=cuda_device, dtype=torch.bfloat16)
    _, grads = with_grads(chunk_decay_attention, xs, cots)
    xs[1] = xs[1].float()
    _, want = with_grads(chunk_decay_attention, xs, cots)
    assert grads[1].dtype == torch.bfloat16 and torch.equal(grads[1], want[1].bfloat16())


def test_offsets_beyond_32_bits_are_held_inside_too(cuda_device):
    from gla_jax_b200 import check_device, chunk_decay_attention_packed
    from gla_jax_b200._lib import GlaError
    xs, _ = packed(cuda_device, 3, 600, 2, 1, 64, 64, torch.bfloat16)
    check_device()
    for offsets in ([0, 2 ** 32 + 100, 400, 600], [0, 100, -2 ** 32 + 300, 600], [0, 100, 400, 2 ** 40 + 600]):
        want = chunk_decay_attention_packed(*xs, torch.tensor(held_inside(offsets, 600), device=cuda_device))
        check_device()
        got = chunk_decay_attention_packed(*xs, torch.tensor(offsets, device=cuda_device))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        with pytest.raises(GlaError):
            check_device()


@pytest.mark.parametrize("rate", [0.02, 0.3, 0.45])
@pytest.mark.parametrize("D", [64, 128])
def test_large_products_under_decay(cuda_device, rate, D):
    """Scores up to 2^35 and products of values and cotangents up to 2^45: nothing between the inputs and the results, the gates'
    gradient of their product among them, may overflow."""
    from gla_jax_b200 import chunk_decay_attention
    xs = make(cuda_device, 1, 260, 2, 2, D, D, torch.bfloat16, torch.float32)
    xs[1] = torch.full_like(xs[1], -rate)
    xs[2], xs[3], xs[4] = xs[2] * 2.0 ** 20, xs[3] * 2.0 ** 17, xs[4] * 2.0 ** 14
    cots = [torch.randn_like(xs[0]), torch.randn_like(xs[2]) * 2.0 ** 20]
    got, grads = with_grads(chunk_decay_attention, xs, cots)
    check(xs, cots, got, grads, torch.bfloat16, torch.float32, rate)


@pytest.mark.parametrize("shift", [-3.0, 0.0, 3.0])
@pytest.mark.parametrize("size", [(2, 250, 2, 2, 64, 64), (1, 900, 4, 2, 128, 32), (1, 333, 2, 1, 24, 200)])
def test_float32_gates_gradient_under_sharp_gates(cuda_device, size, shift):
    """A gate's gradient is about the tokens that it weighs, however many others there are: pairs inside a chunk of 32 are summed as
    they are, and the sums of what comes from outside a chunk, each of its own size, are off by some 2^-23 of theirs: 2^-20 of the
    norm for up to 28 chunks, whose errors fall either way."""
    from gla_jax_b200 import chunk_decay_attention
    xs = make(cuda_device, *size, torch.float32, torch.float32, seed=21, shift=shift)
    gen = torch.Generator(device=cuda_device).manual_seed(22)
    cots = [torch.randn(x.shape, generator=gen, device=cuda_device) for x in (xs[0], xs[2])]
    _, want = with_grads(recurrence, [x.double() for x in xs], [c.double() for c in cots])
    _, got = with_grads(chunk_decay_attention, xs, cots)
    for b in range(size[0]):
        for h in range(size[2]):
            err = (got[1][b, :, h].double() - want[1][b, :, h]).norm() / want[1][b, :, h].norm()
            assert err <= 2.0 ** -20, (b, h, err.item())


def test_float32_packed_gates_gradient_under_sharp_gates(cuda_device):
    """The same for packed sequences, which are cut at cells of the axis, and whose chunks start at their first token."""
    from gla_jax_b200 import chunk_decay_attention_packed
    lens = [5, 0, 470, 1, 33, 0, 600, 64]
    T = sum(lens) + 9
    xs, cots = packed(cuda_device, len(lens), T, 2, 1, 64, 64, torch.float32, seed=23)
    xs[1] = xs[1] - 2.0
    cu = [0, *torch.tensor(lens).cumsum(0).tolist()]
    _, got = with_grads(lambda *a: chunk_decay_attention_packed(*a, torch.tensor(cu, device=cuda_device)), xs, cots)
    for s, (a, b) in enumerate(zip(cu, cu[1:])):
        if a == b:
            continue
        one = [xs[0][s:s + 1], *(x[None, a:b] for x in xs[1:])]
        _, want = with_grads(recurrence, [x.double() for x in one], [cots[0][s:s + 1].double(), cots[1][None, a:b].double()])
        err = (got[1][a:b].double() - want[1][0]).norm() / want[1].norm()
        assert err <= 2.0 ** -20, (s, err.item())
    assert (got[1][cu[-1]:] == 0).all()


@pytest.mark.parametrize("size", [(1, 3000, 2, 2, 256, 64), (2, 1500, 40, 40, 64, 136), (1, 700, 1, 1, 136, 256), (1, 3000, 2, 2, 128, 64),
                                  (2, 1500, 40, 40, 128, 128)])
def test_gates_gradient_far_from_the_end(cuda_device, size):
    """A cotangent of the final state reaches the gates of the last few tokens only, when memories are short: what the others get
    besides is the error of the sum that starts at <S_T, dS_T>, whose parts are held in two bf16 planes and more (2^-16 each)."""
    from gla_jax_b200 import chunk_decay_attention
    xs = make(cuda_device, *size, torch.bfloat16, torch.bfloat16, seed=24, shift=0.0)
    cots = [torch.randn_like(xs[0]), torch.zeros_like(xs[2])]
    _, got = with_grads(chunk_decay_attention, xs, cots)
    up = [x.double().requires_grad_(i == 1) for i, x in enumerate(xs)]
    hf, _ = recurrence(*up)
    want = torch.autograd.grad(hf, up[1], cots[0].double())[0]
    far = got[1][:, : size[1] - 300].double()
    assert want[:, : size[1] - 300].abs().max() < 1e-9
    assert far.abs().max() <= 2.0 ** -13 * want.abs().max(), (far.abs().max().item(), want.abs().max().item())


@pytest.mark.parametrize("dtype,D,packs", [(torch.float32, 64, False), (torch.float32, 64, True), (torch.bfloat16, 136, True), (torch.bfloat16, 64, True)])
def test_backward_in_a_graph_beside_another_stream(cuda_device, dtype, D, packs):
    """Kernels that run beside others inside a call: captured, replayed with new inputs while another stream is at work."""
    from gla_jax_b200 import chunk_decay_attention, chunk_decay_attention_packed
    T = 700
    cu = torch.tensor([0, 300, 301, 640], dtype=torch.int32, device=cuda_device)
    sets = []
    for seed in (31, 32):
        if packs:
            sets.append(packed(cuda_device, 3, T, 2, 1, D, D, dtype, seed=seed))
        else:
            xs = make(cuda_device, 2, T, 2, 1, D, D, dtype, dtype, seed=seed)
            sets.append((xs, [torch.randn_like(xs[0]), torch.randn_like(xs[2])]))
    f = (lambda *a: chunk_decay_attention_packed(*a, cu)) if packs else chunk_decay_attention
    leaves, cots = [x.clone().requires_grad_(True) for x in sets[0][0]], [c.clone() for c in sets[0][1]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(f(*leaves), leaves, cots)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = f(*leaves)
        grads = torch.autograd.grad(outs, leaves, cots)
    want, gw = with_grads(f, *sets[1])
    with torch.no_grad():
        for a, b in zip([*leaves, *cots], [*sets[1][0], *sets[1][1]]):
            a.copy_(b)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            other, go = with_grads(f, *sets[1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([*outs, *grads], [*want, *gw]))
        assert all(torch.equal(a, b) for a, b in zip([*other, *go], [*want, *gw]))


@pytest.mark.parametrize("size", [(2, 84, 3, 3, 8, 128), (3, 557, 2, 2, 32, 32), (1, 841, 1, 1, 80, 32), (2, 112, 3, 3, 112, 32), (1, 274, 2, 1, 24, 32)])
def test_bf16_gradients_of_few_terms(cuda_device, size):
    """Sums of few terms under sharp gates, where a term rounded to bf16 shows: with the gates' gradient every operand is in two
    planes, and the one rounding is the result's."""
    from gla_jax_b200 import chunk_decay_attention
    for seed in range(12):
        xs = make(cuda_device, *size, torch.bfloat16, torch.bfloat16, seed=seed)
        gen = torch.Generator(device=cuda_device).manual_seed(seed)
        u = torch.rand(xs[1].shape, generator=gen, device=cuda_device)
        xs[1] = (-u * 0.3, -u * 5.0, torch.where(u < 0.5, 0.0, -3.0 * u), torch.where(u < 0.05, -1e4, -0.1 * u))[seed % 4].contiguous()
        cots = [torch.randn(x.shape, generator=gen, device=cuda_device).to(x.dtype) for x in (xs[0], xs[2])]
        got, grads = with_grads(chunk_decay_attention, xs, cots)
        check(xs, cots, got, grads, torch.bfloat16, torch.bfloat16, (size, seed))


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 136)])
def test_outputs_before_a_gate_that_is_not_a_number(cuda_device, dtype, D):
    from gla_jax_b200 import chunk_decay_attention
    xs = make(cuda_device, 1, 200, 2, 2, D, D, dtype, dtype)
    want = chunk_decay_attention(*xs)
    for t in (1, 46, 47, 63, 64, 130):
        ys = [x.clone() for x in xs]
        ys[1][0, t, 0] = math.nan
        hf, out = chunk_decay_attention(*ys)
        # (the weights of a chunk are made in another way where its sums are not finite: a rounding of scores and result may differ)
        unit = want[1][:, :t].double().abs() + want[1][:, :t].double().abs().mean()
        assert ((out[:, :t].double() - want[1][:, :t].double()).abs() <= (2.0 ** -5 if dtype == torch.bfloat16 else 2.0 ** -16) * unit).all(), t
        assert torch.equal(out[:, :, 1], want[1][:, :, 1]) and torch.equal(hf[:, 1], want[0][:, 1])
        assert torch.isnan(out[:, t:, 0]).all() and torch.isnan(hf[:, 0]).all()


def test_gates_gradient_over_a_long_uncut_sequence(cuda_device):
    """80 sequences, so that none is cut, of 16384 tokens.  The running sum adds up the errors of its terms: 2^-17 of each from operands
    in two planes, falling either way, the terms being of the gradient's own size: 2^-17 sqrt(16384) = 2^-10 of its norm, whatever
    the gates' memory."""
    from gla_jax_b200 import chunk_decay_attention
    T, D = 16384, 64
    xs = make(cuda_device, 80, T, 1, 1, D, D, torch.bfloat16, torch.bfloat16, seed=41, shift=5.0)
    gen = torch.Generator(device=cuda_device).manual_seed(42)
    cots = [torch.randn(x.shape, generator=gen, device=cuda_device).to(x.dtype) for x in (xs[0], xs[2])]
    _, got = with_grads(chunk_decay_attention, xs, cots)
    for s in (0, 79):
        one = [x[s:s + 1].double().requires_grad_(i == 1) for i, x in enumerate(xs)]
        want = torch.autograd.grad(recurrence(*one), one[1], [c[s:s + 1].double() for c in cots])[0][0, :, 0]
        for part in (slice(0, T // 4), slice(T - T // 4, T), slice(0, T)):
            err = (got[1][s, part, 0].double() - want[part]).norm() / want[part].norm()
            assert err <= 2.0 ** -10, (s, part, err.item())


@pytest.mark.parametrize("size", [(1, 700, 2, 2, 256, 64), (2, 300, 2, 1, 64, 136), (1, 900, 1, 1, 136, 256), (3, 500, 40, 40, 128, 136),
                                  (1, 700, 2, 2, 128, 128)])
def test_bf16_states_leave_with_their_own_rounding(cuda_device, size):
    """The state is summed from terms in two planes and more (2^-16 each), so that what it is off by as it leaves in bf16 is its
    rounding: that of the exact state, but for those that fall the other way."""
    from gla_jax_b200 import chunk_decay_attention
    xs = make(cuda_device, *size, torch.bfloat16, torch.bfloat16, seed=51, shift=4.0)
    hf, _ = chunk_decay_attention(*xs)
    want, _ = recurrence(*(x.double() for x in xs))
    own = (want.bfloat16().double() - want).norm()
    assert (hf.double() - want).norm() <= 1.05 * own, ((hf.double() - want).norm() / want.norm()).item()
