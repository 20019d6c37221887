"""Linear attention with one decay per head, its single-token step, and beam search over recurrent states, as calls that
users make of them: sizes, inputs, one pass each, the same in plain torch operations, and the definition in 64 bits.

``own`` selects the calls of ``gla_jax_b200`` (true) or the plain form (false).  Queries, values and states are N(0, 1), keys
N(0, 1 / Dk).  Decays are either one constant per head ("head": memories of 32 tokens up to 4096) or one per token and head
("token": log_sigmoid(shift + N(0, 1)), shift 5 for soft gates, 0 for sharp ones), the latter in the type of the data, as the
projection that makes them gives them, and with a gradient.
"""
import math
import random

import torch
import torch.nn.functional as F

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f32": 4}


def listed():
    return [
        # training, README shape of this repository: constant decays per head
        dict(name="train_readme", op="attend", dtype="bf16", B=4, T=4096, H=6, Hk=6, Dk=128, Dv=128, nseq=0, decay="head", shift=5.0, grad=True, state="bf16"),
        # training on one long document per GPU: few heads, a very long time axis; the largest call
        dict(name="train_long_context", op="attend", dtype="bf16", B=1, T=131072, H=8, Hk=8, Dk=128, Dv=128, nseq=0, decay="head", shift=5.0, grad=True, state="bf16"),
        # training on documents of different lengths packed on one axis, gates from the data, keys and queries shared by four heads
        dict(name="train_packed_shared", op="attend", dtype="bf16", B=1, T=8191, H=16, Hk=4, Dk=128, Dv=64, nseq=11, decay="token", shift=5.0, grad=True, state="bf16"),
        # a correctness run in full precision: small enough that latency and launches count
        dict(name="check_f32", op="attend", dtype="f32", B=2, T=250, H=2, Hk=2, Dk=64, Dv=64, nseq=0, decay="token", shift=0.0, grad=True, state="f32"),
        # serving: the prompt of one request, forward only, the state kept in float32 for the steps that follow
        dict(name="prefill_prompt", op="attend", dtype="bf16", B=1, T=1155, H=16, Hk=16, Dk=128, Dv=128, nseq=0, decay="token", shift=5.0, grad=False, state="f32"),
        # serving: one token of one request, and of a batch of requests
        dict(name="step_one", op="step", dtype="bf16", N=1, K=1, H=8, Hk=8, Dk=64, Dv=64, shift=5.0, beams=False),
        dict(name="step_batch", op="step", dtype="bf16", N=32, K=1, H=16, Hk=16, Dk=128, Dv=128, shift=5.0, beams=False),
        # serving: one token of every beam, each of which goes on from the state of its parent
        dict(name="step_beams", op="step", dtype="bf16", N=16, K=4, H=16, Hk=4, Dk=128, Dv=64, shift=5.0, beams=True),
        # beam search: a single request over a small vocabulary of odd size, and a batch over a large one
        dict(name="select_one", op="select", dtype="f32", N=1, K=4, V=32001, M=4, finished=False),
        dict(name="select_batch", op="select", dtype="bf16", N=64, K=8, V=128000, M=16, finished=True),
        # beam search: states of all layers moved to where their beams went
        dict(name="reorder_small", op="reorder", dtype="f32", N=1, K=5, layers=3, H=4, D=64),
        dict(name="reorder_layers", op="reorder", dtype="f32", N=16, K=4, layers=12, H=16, D=128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above."""
    op = rng.choice(["attend"] * 5 + ["step", "step", "select", "select", "reorder"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if op == "attend":
        Dk, Dv = rng.choice([32, 64, 64, 128, 128, 128, 80, 256]), rng.choice([32, 64, 64, 128, 128, 128, 96, 256])
        Hk, share = rng.randint(1, 8), rng.choice([1, 1, 1, 2, 3, 4])
        H, grad = Hk * share, rng.random() < 0.6
        # token-heads of the pass: a few tokens up to a training batch
        most = (16 << 10) if dtype == "f32" else (128 << 10) if max(Dk, Dv) > 128 else (384 << 10)
        th = _log_int(rng, 64, most)
        B = _log_int(rng, 1, 12)
        nseq = rng.choice([0, 0, rng.randint(1, 24)])
        T = max(1, th // (H * (1 if nseq else B)))
        if nseq:
            B, T = 1, max(T, 2 * nseq)
        decay = rng.choice(["head", "token"])
        state = "f32" if dtype == "f32" or not grad else "bf16"
        return dict(op=op, dtype=dtype, B=B, T=T, H=H, Hk=Hk, Dk=Dk, Dv=Dv, nseq=nseq, decay=decay,
                    shift=rng.choice([5.0, 5.0, 2.0, 0.0]), grad=grad, state=state)
    if op == "step":
        Hk, K = rng.randint(1, 16), rng.choice([1, 2, 3, 4, 5, 8])
        return dict(op=op, dtype=dtype, N=_log_int(rng, 1, 128) // K + 1, K=K, H=Hk * rng.choice([1, 1, 2]), Hk=Hk,
                    Dk=rng.choice([32, 64, 128, 128, 256, 80]), Dv=rng.choice([32, 64, 128, 128, 256, 96]),
                    shift=rng.choice([5.0, 2.0, 0.0]), beams=K > 1)
    if op == "select":
        K = rng.choice([1, 2, 3, 4, 5, 8, 16])
        V = _log_int(rng, 64, 200000)
        N = max(1, min(96, _log_int(rng, 1 << 10, 48 << 20) // (K * V)))
        return dict(op=op, dtype=dtype, N=N, K=K, V=V, M=min(32, K * rng.choice([1, 2, 2])), finished=rng.random() < 0.5)
    return dict(op=op, dtype=dtype, N=_log_int(rng, 1, 24), K=rng.choice([2, 3, 4, 5, 8]), layers=rng.randint(1, 12), H=rng.randint(1, 16),
                D=rng.choice([32, 64, 128]))


def _offsets(T, nseq, seed):
    """nseq lengths that sum to T, none of them round."""
    r = random.Random(seed)
    w = [0.25 + r.random() for _ in range(nseq)]
    cu, at = [0], 0.0
    for x in w:
        at += x
        cu.append(round(at / sum(w) * T))
    cu[-1] = T
    return cu


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, op = _DTYPES[case["dtype"]], case["op"]

    def new(shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    st = dict(case=case)
    if op == "attend":
        B, T, H, Hk, Dk, Dv = (case[x] for x in ("B", "T", "H", "Hk", "Dk", "Dv"))
        lead = () if case["nseq"] else (B,)
        n = case["nseq"] or B
        if case["nseq"]:
            # as a data loader hands them over: on the GPU, with the lengths known to the host as well
            st["cu_host"] = _offsets(T, case["nseq"], seed)
            st["cu"] = torch.tensor(st["cu_host"], dtype=torch.int32, device="cuda")
        if case["decay"] == "head":
            g = -1.0 / torch.logspace(5, 12, H, base=2.0, device="cuda")
        else:
            g = F.logsigmoid(new(lead + (T, H)) + case["shift"]).to(dt)
        sd = _DTYPES[case["state"]]
        st["x"] = [new((n, H, Dk, Dv), sd), g, new(lead + (T, H, Dv), dt), new(lead + (T, Hk, Dk), dt, Dk ** -0.5),
                   new(lead + (T, Hk, Dk), dt)]
        if case["grad"]:
            for i, x in enumerate(st["x"]):
                x.requires_grad_(i != 1 or case["decay"] == "token")
            st["cotangents"] = [new((n, H, Dk, Dv), sd), new(lead + (T, H, Dv), dt)]
    elif op == "step":
        N, K, H, Hk, Dk, Dv = (case[x] for x in ("N", "K", "H", "Hk", "Dk", "Dv"))
        st["state"] = new((N * K, H, Dk, Dv))
        st["x"] = [F.logsigmoid(new((N * K, H)) + case["shift"]), new((N * K, H, Dv), dt), new((N * K, Hk, Dk), dt, Dk ** -0.5),
                   new((N * K, Hk, Dk), dt)]
        st["parents"] = _parents(N, K, gen) if case["beams"] else None
    elif op == "select":
        N, K, V = case["N"], case["K"], case["V"]
        st["logits"] = new((N, K, V), dt, 3.0)
        st["scores"] = -new((N, K)).abs_().mul_(4.0).cumsum(1)
        # one beam in eight has ended
        st["finished"] = torch.rand((N, K), generator=gen, device="cuda") < 0.125 if case["finished"] else None
    else:
        rows = case["N"] * case["K"]
        st["states"] = [new((rows, case["H"], case["D"], case["D"]), dt) for _ in range(case["layers"])]
        st["parents"] = _parents(case["N"], case["K"], gen)
    return st


def _parents(N, K, gen):
    return torch.randint(0, K, (N, K), generator=gen, device="cuda", dtype=torch.int32)


# ---- the framework's calls -----------------------------------------------------------------------------------------------
def _run_own(st):
    import gla_jax_b200 as gla

    case, op = st["case"], st["case"]["op"]
    if op == "step":
        return gla.decay_attention_step(st["state"], *st["x"], parents=st["parents"]), st["state"]
    if op == "select":
        return gla.beam_select(st["logits"], st["scores"], num_select=case["M"], finished=st["finished"])
    if op == "reorder":
        gla.reorder_states(st["states"], st["parents"])
        return st["states"]
    if case["nseq"]:
        hidden, out = gla.chunk_decay_attention_packed(*st["x"], st["cu"])
    else:
        hidden, out = gla.chunk_decay_attention(*st["x"])
    return _with_grads(st, hidden, out)


def _with_grads(st, hidden, out):
    if not st["case"]["grad"]:
        return hidden, out
    leaves = [x for x in st["x"] if x.requires_grad]
    return hidden, out, torch.autograd.grad([hidden, out], leaves, st["cotangents"])


# ---- the plain form -------------------------------------------------------------------------------------------------------
_CHUNK = 128


def _entering(total, add):
    """States after every chunk from zero, by doubling: (B, H, N) log decays in 64 bits, (B, H, N, Dk, Dv) sums."""
    d, n = 1, total.shape[2]
    while d < n:
        add = torch.cat([add[:, :, :d], add[:, :, d:] + torch.exp(total[:, :, d:]).to(add.dtype)[..., None, None] * add[:, :, :-d]], 2)
        total = torch.cat([total[:, :, :d], total[:, :, d:] + total[:, :, :-d]], 2)
        d *= 2
    return add


def _attend(h, g, v, k, q):
    """Dense batch in 32 bits: h (B, H, Dk, Dv), g (B, T, H), v (B, T, H, Dv), k and q (B, T, Hk, Dk)."""
    B, T, H, _ = v.shape
    share = H // k.shape[2]
    h, v, k, q = h.float(), v.float(), k.float().repeat_interleave(share, 2), q.float().repeat_interleave(share, 2)
    C = min(_CHUNK, T)
    pad = -T % C
    g, v, k, q = F.pad(g.double(), (0, 0, 0, pad)), F.pad(v, (0, 0, 0, 0, 0, pad)), F.pad(k, (0, 0, 0, 0, 0, pad)), F.pad(q, (0, 0, 0, 0, 0, pad))
    N = (T + pad) // C
    lam = g.view(B, N, C, H).permute(0, 3, 1, 2).cumsum(3)                        # running sums in 64 bits
    v, k, q = (x.view(B, N, C, H, -1).permute(0, 3, 1, 2, 4) for x in (v, k, q))  # (B, H, N, C, D)
    later = torch.ones(C, C, dtype=torch.bool, device=v.device).triu(1)
    w = torch.exp((lam[..., :, None] - lam[..., None, :]).masked_fill(later, -math.inf)).float()
    last = lam[..., -1]
    add = (k * torch.exp(last[..., None] - lam).float()[..., None]).transpose(-1, -2) @ v
    first = add[:, :, :1] + torch.exp(last[:, :, :1]).float()[..., None, None] * h[:, :, None]
    after = _entering(last, torch.cat([first, add[:, :, 1:]], 2))
    before = torch.cat([h[:, :, None], after[:, :, :-1]], 2)
    out = ((q @ k.transpose(-1, -2)) * w) @ v + torch.exp(lam).float()[..., None] * (q @ before)
    return after[:, :, -1], out.permute(0, 2, 3, 1, 4).reshape(B, N * C, H, -1)[:, :T]


def _run_attend(st):
    case = st["case"]
    h, g, v, k, q = st["x"]
    if case["decay"] == "head":
        g = g.expand(*v.shape[:-1])
    if not case["nseq"]:
        hidden, out = _attend(h, g, v, k, q)
    else:
        # the sequences as rows of one batch, padded with tokens that neither decay nor add
        cu = st["cu"].long()
        length = cu[1:] - cu[:-1]
        most = max(b - a for a, b in zip(st["cu_host"], st["cu_host"][1:]))
        at = torch.arange(most, device="cuda")
        inside = at < length[:, None]
        take = (cu[:-1, None] + at).clamp(max=case["T"] - 1)
        rows = lambda x: torch.where(inside.view(*inside.shape, *([1] * (x.dim() - 1))), x[take], torch.zeros((), dtype=x.dtype, device="cuda"))  # noqa: E731
        hidden, out = _attend(h, rows(g), rows(v), rows(k), rows(q))
        out = out[inside]
    return _with_grads(st, hidden.to(h.dtype), out.to(v.dtype))


def _run_step(st):
    case, state = st["case"], st["state"]
    g, v, k, q = st["x"]
    if st["parents"] is not None:
        row = torch.arange(case["N"], device="cuda")[:, None] * case["K"] + st["parents"]
        state.copy_(state[row.view(-1)])
    share = case["H"] // case["Hk"]
    k, q = k.float().repeat_interleave(share, 1), q.float().repeat_interleave(share, 1)
    state.mul_(torch.exp(g)[..., None, None]).add_(k[..., None] * v.float()[..., None, :])
    return (q[..., None] * state).sum(-2).to(v.dtype), state


def _log_probs(st):
    """(N, K, V) log-probabilities in 64 bits; a beam that has ended goes on with the padding token (0) alone."""
    x = st["logits"].double()
    top = x.amax(-1, keepdim=True)
    p = (x - top) - torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    if st["finished"] is not None:
        pad = torch.full_like(p[0, 0], -math.inf)
        pad[0] = 0.0
        p = torch.where(st["finished"][..., None], pad, p)
    return p


def _run_select(st):
    case = st["case"]
    total = (st["scores"].double()[..., None] + _log_probs(st)).view(case["N"], -1)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, : case["M"]], at[:, : case["M"]]
    return best.float(), at % case["V"], torch.div(at, case["V"], rounding_mode="floor").int()


def _run_reorder(st):
    case = st["case"]
    row = (torch.arange(case["N"], device="cuda")[:, None] * case["K"] + st["parents"]).view(-1)
    return [s.copy_(s[row]) for s in st["states"]]


def run(st):
    if own:
        return _run_own(st)
    return {"attend": _run_attend, "step": _run_step, "select": _run_select, "reorder": _run_reorder}[st["case"]["op"]](st)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------
def work(case):
    op, e = case["op"], _BYTES[case["dtype"]]
    if op == "attend":
        th, tk = 1.0 * case["B"] * case["T"] * case["H"], 1.0 * case["B"] * case["T"] * case["Hk"]
        state = 1.0 * (case["nseq"] or case["B"]) * case["H"] * case["Dk"] * case["Dv"] * _BYTES[case["state"]]
        gate = th * e if case["decay"] == "token" else 4.0 * case["H"]
        # q, k, v and gates in, out; with gradients the cotangents in and a gradient of each input out
        n = e * (2 * th * case["Dv"] + 2 * tk * case["Dk"]) * (2 if case["grad"] else 1) + 2 * state * (2 if case["grad"] else 1)
        n += gate * (2 if case["grad"] and case["decay"] == "token" else 1)
        return {"bytes": n, "flops": th * case["Dk"] * case["Dv"] * (12 if case["grad"] else 4)}
    if op == "step":
        s = 1.0 * case["N"] * case["K"] * case["H"]
        out = s * case["Dv"] * 2 * e + s * 4 + 2.0 * e * case["N"] * case["K"] * case["Hk"] * case["Dk"]
        read = 1 - (1 - 1 / case["K"]) ** case["K"] if case["beams"] else 1.0      # rows that are somebody's parent
        return {"bytes": out + 4 * s * case["Dk"] * case["Dv"] * (1 + read), "flops": 5.0 * s * case["Dk"] * case["Dv"]}
    if op == "select":
        n = 1.0 * case["N"] * case["K"] * case["V"] * (0.875 if case["finished"] else 1)
        return {"bytes": n * e + case["N"] * (4.0 * case["K"] + 16.0 * case["M"]), "flops": 3.0 * n}
    rows, K = case["N"] * case["K"], case["K"]
    moved = (K - 1) / K                                     # rows whose parent is another one
    taken = 1 - (1 - 1 / K) ** (K - 1)                      # rows that another one goes on from
    return {"bytes": rows * (moved + taken) * e * case["layers"] * case["H"] * case["D"] ** 2, "flops": 0.0}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------
def _definition(h, g, v, k, q):
    """One sequence, 64 tokens at a time: h (H, Dk, Dv), g (T, H), the rest (T, H, D), all in 64 bits."""
    outs = []
    for a in range(0, v.shape[0], 64):
        gc, vc, kc, qc = (x[a:a + 64] for x in (g, v, k, q))
        lam = gc.cumsum(0).t()                                                    # (H, C)
        pair = lam[:, :, None] - lam[:, None, :]
        pair = torch.where(torch.ones_like(pair).tril() > 0, pair, torch.full_like(pair, -1e4)).exp()
        score = torch.einsum("ihd,jhd->hij", qc, kc) * pair
        outs.append(torch.einsum("hij,jhe->ihe", score, vc) + torch.einsum("ihd,hde->ihe", qc * lam.t().exp()[..., None], h))
        tail = (lam[:, -1:] - lam).exp().t()[..., None]
        h = h * lam[:, -1].exp()[:, None, None] + torch.einsum("jhd,jhe->hde", kc * tail, vc)
    return h, torch.cat(outs) if outs else torch.zeros_like(v)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "reorder":
        return None
    if case["op"] == "select":
        x = st["logits"].double()
        p = x - torch.logsumexp(x, -1, keepdim=True)
        if st["finished"] is not None:
            p[st["finished"]] = -math.inf
            p[..., 0] = torch.where(st["finished"], torch.zeros_like(p[..., 0]), p[..., 0])
        total = (p + st["scores"].double()[..., None]).flatten(1)
        return total.topk(case["M"], 1).values, None, None
    if case["op"] == "step":
        S = st["state"].double()
        g, v, k, q = (x.double() for x in st["x"])
        rep = case["H"] // case["Hk"]
        if st["parents"] is not None:
            S = torch.stack([S[n * case["K"] + p] for n in range(case["N"]) for p in st["parents"][n].tolist()])
        S = S * g.exp()[..., None, None] + torch.einsum("bhd,bhe->bhde", k.repeat_interleave(rep, 1), v)
        return torch.einsum("bhd,bhde->bhe", q.repeat_interleave(rep, 1), S), S
    leaves = [x.detach().double().requires_grad_(x.requires_grad) for x in st["x"]]
    h, g, v, k, q = leaves
    rep = case["H"] // case["Hk"]
    if case["decay"] == "head":
        g = g.expand(*v.shape[:-1])
    k, q = k.repeat_interleave(rep, -2), q.repeat_interleave(rep, -2)
    if case["nseq"]:
        cu = st["cu_host"]
        got = [_definition(h[s], *(x[a:b] for x in (g, v, k, q))) for s, (a, b) in enumerate(zip(cu, cu[1:]))]
        hidden, out = torch.stack([x[0] for x in got]), torch.cat([x[1] for x in got])
    else:
        # the batch as more heads
        B, T, H, Dv = v.shape
        flat = lambda x: x.transpose(0, 1).reshape(T, B * H, *x.shape[3:])  # noqa: E731
        hidden, out = _definition(h.flatten(0, 1), flat(g), flat(v), flat(k), flat(q))
        hidden, out = hidden.view(h.shape), out.view(T, B, H, Dv).transpose(0, 1)
    if not case["grad"]:
        return hidden, out
    grads = torch.autograd.grad([hidden, out], [x for x in leaves if x.requires_grad], [c.double() for c in st["cotangents"]])
    return hidden.detach(), out.detach(), grads
