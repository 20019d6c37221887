"""Beam search over recurrent states: selection, moving of states, steps that follow parents, and a whole search."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def selected(logits, scores, M, finished=None, pad=0):
    """The definition in 64 bits: a stable sort of all totals."""
    x = logits.double().nan_to_num(nan=-math.inf, posinf=3.4028234663852886e38, neginf=-math.inf)
    top = x.amax(-1, keepdim=True)
    # (rows padded to one alignment: torch's sum of a row goes by its address, and equal rows have to have equal sums)
    e = torch.nn.functional.pad((x - top).exp(), (0, -x.shape[-1] % 64))
    p = (x - top) - e.sum(-1, keepdim=True).log()
    p = torch.where(top > -math.inf, p, torch.full_like(p, -math.inf))
    if finished is not None:
        only = torch.full_like(p, -math.inf)
        only[..., pad] = 0.0
        p = torch.where(finished[..., None], only, p)
    total = (scores.double()[..., None] + p).nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf).flatten(1)
    best, at = total.sort(dim=1, descending=True, stable=True)
    V = logits.shape[-1]
    return best[:, :M], at[:, :M] % V, at[:, :M] // V


def same(got, want):
    scores, tokens, parents = got
    assert torch.equal(tokens, want[1]) and torch.equal(parents.long(), want[2])
    fin = torch.isfinite(want[0])
    assert torch.equal(torch.isfinite(scores), fin)
    # the total rounded once, and a logarithm of a float32 sum of exponentials: 2^-24 of the total and 2^-20
    assert ((scores.double() - want[0])[fin].abs() <= 2.0 ** -24 * want[0][fin].abs() + 2.0 ** -20).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,K,V,M", [(1, 1, 1, 1), (2, 3, 2, 6), (3, 4, 17, 8), (2, 5, 4095, 5), (1, 4, 4097, 32), (3, 2, 33333, 4),
                                     (2, 32, 1000, 32), (1, 8, 100003, 16), (70, 2, 777, 4)])
def test_selection(cuda_device, N, K, V, M, dtype):
    from gla_jax_b200 import beam_select
    gen = torch.Generator(device=cuda_device).manual_seed(N * V + M)
    logits = (3 * torch.randn(N, K, V, generator=gen, device=cuda_device)).to(dtype)
    scores = -10 * torch.rand(N, K, generator=gen, device=cuda_device)
    same(beam_select(logits, scores, M), selected(logits, scores, M))
    if K > 1 and V > 2:
        fin = torch.rand(N, K, generator=gen, device=cuda_device) < 0.5
        same(beam_select(logits, scores, M, finished=fin, pad_token=2), selected(logits, scores, M, fin, 2))
        scores[:, 1:] = -math.inf                                    # the first token of a search
        same(beam_select(logits, scores, M), selected(logits, scores, M))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_selection_of_ties_masks_and_odd_values(cuda_device, dtype):
    from gla_jax_b200 import beam_select
    N, K, V, M = 2, 3, 9001, 12
    z = torch.zeros(N, K, V, device=cuda_device, dtype=dtype)
    s = torch.zeros(N, K, device=cuda_device)
    low = torch.finfo(dtype).min
    ramp = torch.arange(V, device=cuda_device, dtype=torch.float32).to(dtype).expand(N, K, V).contiguous()
    late = torch.full_like(z, -math.inf)
    late[..., 5000:] = 1.0
    one = torch.full_like(z, -math.inf)
    one[:, 1, 77] = 3.0
    lowest = torch.full_like(z, low)
    lowest[..., 8000] = 0
    odd = torch.randn(N, K, V, device=cuda_device).to(dtype)
    odd[0, 0, 5], odd[0, 1, 3], odd[1, 2, 8999], odd[1, 0] = math.nan, math.inf, math.inf, math.nan
    steps = (torch.randn(N, K, V, device=cuda_device) * 2).round().to(dtype)                # many equal logits
    sign = z.clone()
    sign[..., ::2] = -0.0
    for x in (z, ramp, ramp.flip(-1), late, one, lowest, odd, steps, sign, torch.full_like(z, -math.inf), torch.full_like(z, math.nan)):
        for m in (1, M, 32):
            same(beam_select(x, s, m), selected(x, s, m))
    s2 = torch.tensor([[0.0, -math.inf, math.nan], [-math.inf] * 3], device=cuda_device)
    want = selected(steps, s2.nan_to_num(nan=-math.inf, neginf=-math.inf), M)
    same(beam_select(steps, s2, M), want)
    # rows that start anywhere
    big = torch.randn(N * K * V + 3, device=cuda_device).to(dtype)
    for off in (1, 3):
        x = big[off:off + N * K * V].view(N, K, V)
        same(beam_select(x, s, M), selected(x, s, M))


@pytest.mark.parametrize("N,K", [(1, 1), (3, 4), (2, 32), (5, 7)])
def test_reorder(cuda_device, N, K):
    from gla_jax_b200 import reorder_states
    gen = torch.Generator(device=cuda_device).manual_seed(K)
    for parents in (torch.randint(0, K, (N, K), generator=gen, device=cuda_device), torch.arange(K, device=cuda_device).roll(1).expand(N, K).contiguous(),
                    torch.arange(K, device=cuda_device).expand(N, K), torch.full((N, K), K - 1, device=cuda_device)):
        row = (torch.arange(N, device=cuda_device)[:, None] * K + parents).flatten()
        states = [torch.randn(N * K, 2, 64, 64, device=cuda_device), torch.randn(N * K, 3, 5, device=cuda_device).bfloat16(),
                  torch.randint(0, 9, (N * K, 7), device=cuda_device), torch.randint(0, 2, (N * K,), device=cuda_device).bool(),
                  torch.randn(N * K + 1, 5, device=cuda_device)[1:], torch.randn(N * K, 0, device=cuda_device)]
        states += [torch.randn(N * K, 33 + i, device=cuda_device) for i in range(70)]       # more than a launch takes
        want = [s[row] for s in states]
        reorder_states(states, parents.to(torch.int32))
        for a, b in zip(states, want):
            assert torch.equal(a, b)
    one = torch.randn(N * K, 12, device=cuda_device)
    want = one[row]
    reorder_states(one, parents)                                                            # int64
    assert torch.equal(one, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,K,H,Hk,Dk,Dv", [(3, 1, 2, 2, 64, 64), (2, 4, 4, 2, 128, 64), (1, 5, 2, 1, 80, 96), (2, 8, 2, 2, 128, 128),
                                            (1, 32, 1, 1, 256, 40), (1, 16, 2, 2, 256, 256)])
def test_steps_follow_parents(cuda_device, N, K, H, Hk, Dk, Dv, dtype):
    from gla_jax_b200 import decay_attention_step, decode_step
    gen = torch.Generator(device=cuda_device).manual_seed(Dk + K)
    n = lambda *s: torch.randn(*s, generator=gen, device=cuda_device)  # noqa: E731
    B = N * K
    parents = torch.randint(0, K, (N, K), generator=gen, device=cuda_device, dtype=torch.int32)
    row = (torch.arange(N, device=cuda_device)[:, None] * K + parents).flatten()
    state, g = n(B, H, Dk, Dv), -n(B, H).abs()
    v, k, q = n(B, H, Dv).to(dtype), n(B, Hk, Dk).to(dtype), n(B, Hk, Dk).to(dtype)
    a, b = state.clone(), state[row].contiguous()
    o1 = decay_attention_step(a, g, v, k, q, parents=parents)
    o2 = decay_attention_step(b, g, v, k, q)
    assert torch.equal(a, b)
    # the sums over features are added in another order: 16 additions of Dk terms
    unit = (q.float().abs().repeat_interleave(H // Hk, 1)[..., None] * b.abs()).sum(-2)
    tol = 2.0 ** -19 + (2.0 ** -7 if dtype == torch.bfloat16 else 0)
    assert ((o1.float() - o2.float()).abs() <= tol * unit).all()
    if Dk == Dv and Hk == H:
        f = -n(B, H, Dk).abs()
        a, b = state.clone(), state[row].contiguous()
        o1, o2 = decode_step(a, f, v, k, q, parents=parents), decode_step(b, f, v, k, q)
        assert torch.equal(a, b) and ((o1.float() - o2.float()).abs() <= tol * (q.float().abs()[..., None] * b.abs()).sum(-2)).all()


def test_bad_parents_are_reported(cuda_device):
    from gla_jax_b200 import check_device, decay_attention_step, reorder_states
    from gla_jax_b200._lib import GlaError
    check_device()
    bad = torch.tensor([[0, 7], [-4, 1]], dtype=torch.int32, device=cuda_device)
    x = torch.randn(4, 2, 64, 64, device=cuda_device)
    want = x[torch.tensor([0, 1, 2, 3], device=cuda_device)].clone()
    reorder_states(x, bad)                                       # held inside: 7 is 1, -4 is 0
    assert torch.equal(x, want)
    with pytest.raises(GlaError, match="2 parent"):
        check_device()
    z = torch.zeros(4, 2, 64, device=cuda_device)
    decay_attention_step(x, torch.zeros(4, 2, device=cuda_device), z, z, z, parents=bad)
    assert torch.equal(x, want)
    with pytest.raises(GlaError, match="2 parent"):
        check_device()
    check_device()


def test_a_search(cuda_device):
    """A prompt, its state given to all beams, and ten tokens of search, against the same in 64 bits."""
    from gla_jax_b200 import beam_select, chunk_decay_attention, decay_attention_step, reorder_states
    gen = torch.Generator(device=cuda_device).manual_seed(5)
    n = lambda *s: torch.randn(*s, generator=gen, device=cuda_device)  # noqa: E731
    N, K, H, D, V, T, steps, eos = 2, 4, 2, 32, 61, 19, 10, 3
    emb, wo = n(V, H, 3, D) * 0.5, n(H * D, V) * 0.6
    g = torch.tensor([-0.1, -0.6], device=cuda_device)
    prompt = torch.randint(4, V, (N, T), generator=gen, device=cuda_device)
    x = emb[prompt]
    h0 = torch.zeros(N, H, D, D, device=cuda_device)
    state, out = chunk_decay_attention(h0, g, *(x[:, :, :, i] for i in range(3)))
    state64 = torch.zeros(N, H, D, D, device=cuda_device, dtype=torch.float64)
    for t in range(T):
        state64 = g.double().exp()[:, None, None] * state64 + x[:, t, :, 1, :, None].double() * x[:, t, :, 0, None, :].double()
    state, state64 = state.repeat_interleave(K, 0), state64.repeat_interleave(K, 0)
    history = torch.zeros(N * K, steps, dtype=torch.int64, device=cuda_device)
    history64 = history.clone()
    scores = torch.full((N, K), -math.inf, device=cuda_device)
    scores[:, 0] = 0
    scores64, tokens64 = scores.double(), None
    tokens = prompt[:, -1:].expand(N, K)
    tokens64 = tokens
    parents = torch.arange(K, device=cuda_device, dtype=torch.int32).expand(N, K).contiguous()
    parents64 = parents.long()
    finished = finished64 = torch.zeros(N, K, dtype=torch.bool, device=cuda_device)
    base = torch.arange(N, device=cuda_device)[:, None] * K
    for t in range(steps):
        e = emb[tokens.flatten()]
        out = decay_attention_step(state, g.expand(N * K, H), e[:, :, 0], e[:, :, 1], e[:, :, 2], parents=parents)
        scores, tokens, parents = beam_select((out.flatten(1) @ wo).view(N, K, V), scores, finished=finished, pad_token=eos)
        finished = finished.gather(1, parents.long()) | (tokens == eos)
        reorder_states(history, parents)
        history[:, t] = tokens.flatten()
        e = emb[tokens64.flatten()].double()
        state64 = state64[(base + parents64).flatten()]
        state64 = g.double().exp()[:, None, None] * state64 + e[:, :, 1, :, None] * e[:, :, 0, None, :]
        o = (e[:, :, 2, :, None] * state64).sum(-2)
        scores64, tokens64, parents64 = selected((o.flatten(1) @ wo.double()).view(N, K, V), scores64, K, finished64, eos)
        finished64 = finished64.gather(1, parents64) | (tokens64 == eos)
        history64 = history64[(base + parents64).flatten()]
        history64[:, t] = tokens64.flatten()
    assert torch.equal(history, history64)
    torch.testing.assert_close(scores.double(), scores64, rtol=1e-4, atol=1e-4)


def test_in_a_graph(cuda_device):
    from gla_jax_b200 import beam_select, decay_attention_step, reorder_states
    N, K, V = 2, 4, 5000
    logits, scores = torch.randn(N, K, V, device=cuda_device), torch.randn(N, K, device=cuda_device)
    state, extra = torch.randn(N * K, 2, 64, 64, device=cuda_device), torch.randn(N * K, 40, device=cuda_device)
    x = torch.randn(N * K, 2, 64, device=cuda_device)

    def once():
        s, t, p = beam_select(logits, scores)
        reorder_states([extra], p)
        return s, t, p, decay_attention_step(state, x[..., 0], x, x, x, parents=p)

    once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    logits.copy_(torch.randn_like(logits))
    a, b = state.clone(), extra.clone()
    graph.replay()
    s1, e1, g1 = state.clone(), extra.clone(), [y.clone() for y in got]
    state.copy_(a)
    extra.copy_(b)
    for y, z in zip(once(), g1):
        assert torch.equal(y, z)
    assert torch.equal(state, s1) and torch.equal(extra, e1)


def test_refusals(cuda_device):
    from gla_jax_b200 import beam_select, reorder_states
    x, s = torch.randn(2, 3, 10, device=cuda_device), torch.randn(2, 3, device=cuda_device)
    for bad in (dict(num_select=0), dict(num_select=33), dict(pad_token=10), dict(finished=torch.zeros(2, 3, device=cuda_device)),
                dict(finished=torch.zeros(2, 2, dtype=torch.bool, device=cuda_device))):
        with pytest.raises(ValueError):
            beam_select(x, s, **bad)
    with pytest.raises(ValueError):
        beam_select(x, s[:1])
    with pytest.raises(TypeError):
        beam_select(x.half(), s)
    with pytest.raises(ValueError):
        beam_select(torch.randn(1, 33, 10, device=cuda_device), torch.randn(1, 33, device=cuda_device))
    p = torch.zeros(2, 3, dtype=torch.int32, device=cuda_device)
    y = torch.randn(6, 8, device=cuda_device)
    with pytest.raises(ValueError, match="overlap"):
        reorder_states([y, y], p)
    with pytest.raises(ValueError, match="rows"):
        reorder_states([y[:5]], p)
    with pytest.raises(ValueError, match="contiguous"):
        reorder_states([y.t()[:6]], p)
    with pytest.raises(TypeError):
        reorder_states([y], p.float())
    with pytest.raises(RuntimeError, match="not differentiable"):
        reorder_states([y.clone().requires_grad_(True)], p)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_selection_where_a_few_threads_hold_all_that_is_large(cuda_device, dtype):
    """Columns laid out as the kernel's threads meet them: the first thirty of 256 hold what is large, so that the bound is low
    and the M largest are found one after the other; and rows of four distinct values."""
    from gla_jax_b200 import beam_select
    N, K, V, M = 1, 2, 60000, 32
    gen = torch.Generator(device=cuda_device).manual_seed(11)
    x = torch.randn(N, K, V, generator=gen, device=cuda_device)
    width = 8 if dtype == torch.bfloat16 else 4
    few = (torch.arange(V, device=cuda_device) // width) % 256 < 30
    logits = torch.where(few, x + 20, x).to(dtype)
    scores = torch.tensor([[-1.0, -1.5]], device=cuda_device)
    same(beam_select(logits, scores, M), selected(logits, scores, M))
    coarse = torch.randint(0, 4, (3, 4, 20000), generator=gen, device=cuda_device).to(dtype)
    flat = torch.tensor([[0.0, 0.0, -1.0, 0.0]], device=cuda_device).expand(3, 4).contiguous()
    # (sums of exponentials of equal counts are not equal to the last bit: the beams are told apart by a whole unit)
    flat = flat - torch.arange(4, device=cuda_device)
    same(beam_select(coarse, flat, M), selected(coarse, flat, M))
    # rising and falling runs: the second largest before, at and behind the largest
    saw = ((torch.arange(20000, device=cuda_device) * 7919) % 251).float().expand(3, 4, 20000).contiguous().to(dtype)
    same(beam_select(saw, flat, M), selected(saw, flat, M))


@pytest.mark.parametrize("D", [32, 256])
def test_decode_steps_of_thirty_two_beams(cuda_device, D):
    from gla_jax_b200 import decode_step
    gen = torch.Generator(device=cuda_device).manual_seed(D)
    n = lambda *s: torch.randn(*s, generator=gen, device=cuda_device)  # noqa: E731
    parents = torch.randint(0, 32, (2, 32), generator=gen, device=cuda_device, dtype=torch.int32)
    row = (torch.arange(2, device=cuda_device)[:, None] * 32 + parents).flatten()
    state, f = n(64, 2, D, D), -n(64, 2, D).abs()
    v, k, q = (n(64, 2, D) for _ in range(3))
    a, b = state.clone(), state[row].contiguous()
    o1, o2 = decode_step(a, f, v, k, q, parents=parents), decode_step(b, f, v, k, q)
    # (the order of up to 256 additions)
    assert torch.equal(a, b) and ((o1 - o2).abs() <= 2.0 ** -16 * (q.abs()[..., None] * b.abs()).sum(-2)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,K,V,M", [(2, 3, 700, 12), (1, 4, 40000, 16), (1, 32, 9000, 32), (3, 1, 5, 4)])
def test_equal_totals_of_unequal_logits(cuda_device, N, K, V, M, dtype):
    """The lowest (beam, token) comes first whatever the logits: where scores leave none of a logit's digits (-1e18 and the type's
    lowest, the usual masks of a score), and where logits differ by less than a total resolves."""
    from gla_jax_b200 import beam_select
    gen = torch.Generator(device=cuda_device).manual_seed(V)
    x = (3 * torch.randn(N, K, V, generator=gen, device=cuda_device)).to(dtype)
    x[..., V // 3] = -math.inf
    for low in (-1e18, torch.finfo(torch.float32).min):
        s = torch.full((N, K), low, device=cuda_device)
        same(beam_select(x, s, M), selected(x, s, M))
        s[:, 0] = 0.0
        few = x.clone()
        few[:, 0, 3:] = -math.inf                           # three tokens of the one beam that counts, the rest from the others
        same(beam_select(few, s, M), selected(few, s, M))
        fin = torch.zeros(N, K, dtype=torch.bool, device=cuda_device)
        fin[:, -1] = True
        same(beam_select(few, s, M, finished=fin, pad_token=2), selected(few, s, M, fin, 2))
    tiny = (torch.arange(V, device=cuda_device) * 1e-25).expand(N, K, V).contiguous().to(dtype)
    s = -torch.arange(K, device=cuda_device).float().expand(N, K).contiguous()
    same(beam_select(tiny, s, M), selected(tiny, s, M))
    # zeros among larger and smaller ones
    some = torch.where(torch.rand(N, K, V, generator=gen, device=cuda_device) < 0.001, x.float().abs(), -x.float().abs().nan_to_num(posinf=1.0)).to(dtype)
    some[torch.rand(N, K, V, generator=gen, device=cuda_device) < 0.5] = 0.0
    same(beam_select(some, s, M), selected(some, s, M))


def test_no_states_to_move(cuda_device):
    from gla_jax_b200 import reorder_states
    parents = torch.tensor([[1, 0]], dtype=torch.int32, device=cuda_device)
    reorder_states([], parents)
    reorder_states((), parents)
    reorder_states([torch.empty(2, 0, device=cuda_device), torch.empty(2, 3, 0, 5, device=cuda_device)], parents)


def test_steps_of_no_requests(cuda_device):
    """The last request of a batch has ended."""
    from gla_jax_b200 import decay_attention_step, decode_step
    state, x = torch.empty(0, 2, 64, 64, device=cuda_device), torch.empty(0, 2, 64, device=cuda_device)
    parents = torch.empty(0, 4, dtype=torch.int32, device=cuda_device)
    assert decode_step(state, x, x, x, x, parents=parents).shape == (0, 2, 64)
    assert decay_attention_step(state, x[..., 0], x, x, x, parents=parents).shape == (0, 2, 64)
    assert decay_attention_step(state, x[..., 0], x, x, x).shape == (0, 2, 64)


def test_states_that_start_anywhere(cuda_device):
    """A contiguous state between multiples of 16 bytes, as a slice of a flat buffer is, is stepped in place like any other."""
    from gla_jax_b200 import decay_attention_step, decode_step
    gen = torch.Generator(device=cuda_device).manual_seed(8)
    n = lambda *s: torch.randn(*s, generator=gen, device=cuda_device)  # noqa: E731
    B, H, D = 6, 2, 64
    parents = torch.tensor([[1, 1, 0], [2, 0, 2]], dtype=torch.int32, device=cuda_device)
    state, v, k, q = n(B, H, D, D), n(B, H, D), n(B, H, D), n(B, H, D)
    for step, g in ((decay_attention_step, -n(B, H).abs()), (decode_step, -n(B, H, D).abs())):
        for par in (None, parents):
            a = state.clone()
            flat = torch.zeros(state.numel() + 2, device=cuda_device)
            b = flat[1:-1].view_as(state).copy_(state)
            assert b.data_ptr() % 16 and b.is_contiguous()
            assert torch.equal(step(a, g, v, k, q, parents=par), step(b, g, v, k, q, parents=par))
            assert torch.equal(a, b) and flat[0] == 0 and flat[-1] == 0


def test_more_rows_than_a_grid_is_high(cuda_device):
    """Batches of more than 65535 (request, head) or (request, beam) pairs equal the halves of them."""
    from gla_jax_b200 import beam_select, decay_attention_step, decode_step
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=gen, device=cuda_device)  # noqa: E731
    B, H, D = 2 * 4120, 16, 32
    for step, K in ((decay_attention_step, 1), (decay_attention_step, 2), (decode_step, 2)):
        keyed = step is decode_step
        state, g = n(B, H, D, D), -n(B, H, *([D] if keyed else [])).abs()
        v, k, q = n(B, H, D), n(B, H, D), n(B, H, D)
        par = torch.randint(0, K, (B // K, K), generator=gen, device=cuda_device, dtype=torch.int32) if K > 1 else None
        a, b = state.clone(), state.clone()
        out = step(a, g, v, k, q, parents=par)
        for s in (slice(0, B // 2), slice(B // 2, B)):
            part = step(b[s], g[s], v[s], k[s], q[s], parents=par[s.start // K:s.stop // K] if K > 1 else None)
            assert torch.equal(part, out[s])
        assert torch.equal(a, b)
    logits, scores = n(35000, 2, 9), n(35000, 2)
    same(beam_select(logits, scores), selected(logits, scores, 2))


def test_bad_parents_of_several_launches_are_counted_once(cuda_device):
    """Tensors of 16-, 4- and 1-byte rows go in launches of their own, and no more than 64 in one."""
    from gla_jax_b200 import check_device, reorder_states
    from gla_jax_b200._lib import GlaError
    check_device()
    bad = torch.tensor([[0, 7], [-4, 1], [1, 0]], dtype=torch.int32, device=cuda_device)
    states = [torch.randn(6, 8, device=cuda_device), torch.randn(6, 5, device=cuda_device), torch.ones(6, 3, device=cuda_device).bool()]
    states += [torch.randn(6, 8, device=cuda_device) for _ in range(70)]
    want = [torch.cat([s[:4], s[5:], s[4:5]]) for s in states]
    reorder_states(states, bad)
    assert all(torch.equal(a, b) for a, b in zip(states, want))
    with pytest.raises(GlaError, match=" 2 parent"):
        check_device()
    check_device()


def _one_part(K, M, V, dtype):
    """Tiles of 4096 logits in a part of a row: 1024 candidates a request are all that there is room for, so that 32 beams with 32
    to select have a single part each."""
    assert 1024 // (K * M) == 1
    return -(-V // 4096)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_selection_one_after_the_other(cuda_device, dtype):
    """A part of many tiles in which thirty of 256 threads hold all that is large: the bound is the lowest there is, and the logits
    that reach it are more than the 1024 that the list holds, so that the M largest are found one after the other."""
    from gla_jax_b200 import beam_select
    N, K, V, M = 2, 32, 60001, 32
    tiles = _one_part(K, M, V, dtype)
    gen = torch.Generator(device=cuda_device).manual_seed(12)
    x = torch.randn(N, K, V, generator=gen, device=cuda_device)
    width = 8 if dtype == torch.bfloat16 else 4
    owner = (torch.arange(V, device=cuda_device) // width) % 256
    few = owner < 30
    # (the bound is the 32nd of the threads' largest, so at most the second of the other threads' largest: below + 10)
    assert tiles > 4 and int(few.sum()) > 1024
    logits = torch.where(few, x.clamp(-4, 4) + 20, x.clamp(-4, 4)).to(dtype)
    scores = -torch.arange(K, device=cuda_device).float().expand(N, K).contiguous()
    same(beam_select(logits, scores, M), selected(logits, scores, M))
    equal = torch.where(few, torch.full_like(x, 3.0), x.clamp(-2, 2)).to(dtype)           # all that is large is equal
    same(beam_select(equal, scores, M), selected(equal, scores, M))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_selection_across_the_tiles_of_a_part(cuda_device, dtype):
    """The two largest of a thread in an earlier, the same and a later tile, equal and unequal, and what else it met below them."""
    from gla_jax_b200 import beam_select
    N, K, V, M = 1, 32, 30011, 32
    assert _one_part(K, M, V, dtype) == 8
    gen = torch.Generator(device=cuda_device).manual_seed(13)
    i = torch.arange(V, device=cuda_device)
    scores = -3.0 * torch.arange(K, device=cuda_device).float().expand(N, K).contiguous()
    noise = torch.rand(N, K, V, generator=gen, device=cuda_device)
    ramp = (i.float() / 64).expand(N, K, V)
    saw = ((i * 7919) % 251).float().expand(N, K, V)
    coarse = torch.randint(0, 4, (N, K, V), generator=gen, device=cuda_device).float()
    cases = [noise, ramp, ramp.flip(-1), saw, saw.flip(-1), coarse]
    # one thread's places (token 4096 t + j of tile t): pairs of tiles hold its largest and second largest, in either order
    for a, b in ((0, 0), (0, 3), (3, 0), (2, 7), (7, 2), (6, 6)):
        for high, low in ((9.0, 8.0), (9.0, 9.0)):
            y = noise.clone()
            y[..., min(4096 * a + 2, V - 2)], y[..., min(4096 * b + 3, V - 1)] = high, low
            y[..., 4096 * 4 + 1] = 7.0
            cases.append(y)
    masked = noise.clone()
    masked[..., : 4096 * 5] = -math.inf
    cases.append(masked)
    for c, x in enumerate(cases):
        x = x.contiguous().to(dtype)
        for m in (M, 1, 5):
            same(beam_select(x, scores, m), selected(x, scores, m))


def test_selection_and_moving_for_no_requests(cuda_device):
    from gla_jax_b200 import beam_select, reorder_states
    scores, tokens, parents = beam_select(torch.empty(0, 4, 50, device=cuda_device), torch.empty(0, 4, device=cuda_device), 3,
                                          finished=torch.empty(0, 4, dtype=torch.bool, device=cuda_device))
    assert scores.shape == tokens.shape == parents.shape == (0, 3) and (scores.dtype, tokens.dtype, parents.dtype) == (torch.float32, torch.int64, torch.int32)
    reorder_states([torch.empty(0, 8, device=cuda_device)], torch.empty(0, 4, dtype=torch.int32, device=cuda_device))
    with pytest.raises(ValueError):
        beam_select(torch.empty(2, 0, 50, device=cuda_device), torch.empty(2, 0, device=cuda_device), 1)
    with pytest.raises(ValueError):
        beam_select(torch.empty(2, 4, 0, device=cuda_device), torch.empty(2, 4, device=cuda_device), 1)
    with pytest.raises(ValueError):
        reorder_states([torch.empty(0, 8, device=cuda_device)], torch.empty(2, 0, dtype=torch.int32, device=cuda_device))
