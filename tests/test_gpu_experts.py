"""gr_route_experts and gr_expert_mlp against float64.

Routing: the same experts as float64 gives, weights to float32 rounding.  The
experts' layers: bounds from float32 sums (K / 8 + 8 units of 2^-24 of the sum of
magnitudes), the gated product's rounding to x's type carried through the down
product, and the result's."""

import pytest
import torch

from tests.test_gpu_fp8_linear import expand, quantise, weights
from vllm_gr_amd import ops

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def route_ref(logits, k, score, bias, groups, top, renorm, scale):
    """Row by row on the CPU in float64."""
    x = logits.double()
    T, E = x.shape
    ids = torch.zeros(T, k, dtype=torch.int32)
    w = torch.zeros(T, k, dtype=torch.float64)
    s = torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, 1)
    for t in range(T):
        st = s[t]
        if score == "softmax" and (x[t] == -float("inf")).all():
            st = torch.zeros(E, dtype=torch.float64)
        c = (st + bias.double() if bias is not None else x[t]).tolist()
        # a NaN after everything, then the larger value, then the lower index
        key = lambda i: (c[i] != c[i], -c[i] if c[i] == c[i] else 0.0, i)
        n = E // groups
        open_ = list(range(E))
        if groups > 1:
            vals = []
            for g in range(groups):
                best = sorted(range(g * n, g * n + n), key=key)[:2 if bias is not None else 1]
                v = sum(c[i] for i in best)
                vals.append((v != v, -v if v == v else 0.0, g))
            kept = {g for _, _, g in sorted(vals)[:top]}
            open_ = [i for i in open_ if i // n in kept]
        pick = sorted(open_, key=key)[:k]
        ids[t] = torch.tensor(pick)
        w[t] = st[pick]
        if renorm:
            tot = w[t].sum()
            w[t] = 0.0 if tot == 0 else w[t] / tot
    return w * scale, ids


CASES = [  # T, E, k, score, bias, groups, top groups, renormalise, scale
    (1, 1, 1, "softmax", False, 1, 1, True, 1.0), (5, 64, 8, "softmax", False, 1, 1, True, 1.0),
    (3, 7, 7, "sigmoid", False, 1, 1, False, 2.5), (33, 60, 6, "softmax", True, 4, 2, False, 1.0),
    (130, 256, 8, "sigmoid", True, 8, 4, True, 2.5), (9, 65, 5, "softmax", True, 1, 1, True, 1.0),
    (7, 1024, 64, "sigmoid", True, 64, 9, True, 1.0), (6, 500, 3, "softmax", False, 5, 1, True, 1.0),
    (11, 8, 4, "sigmoid", True, 8, 4, True, 1.0), (257, 129, 1, "softmax", False, 3, 3, False, 1.0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,score,bias,groups,top,renorm,scale", CASES)
def test_route(device, dtype, T, E, k, score, bias, groups, top, renorm, scale):
    g = torch.Generator().manual_seed(T + E + k)
    wide = (2 * torch.randn(T, E + 3, generator=g)).to(dtype)
    wide[-1, :E // 2] = wide[-1, 0]  # equal logits
    b = 0.1 * torch.randn(E, generator=g) if bias else None
    if bias:
        b[:E // 3] = 0.25  # equal biases
    w, ids = ops.route_experts(wide.to(device)[:, :E], k, score=score, bias=None if b is None else b.to(device),
                               num_groups=groups, top_groups=top, renormalize=renorm, scale=scale)
    rw, rids = route_ref(wide[:, :E], k, score, b, groups, top, renorm, scale)
    assert torch.equal(ids.cpu(), rids)
    assert ((w.cpu().double() - rw).abs() <= rw.abs() * 2.0 ** -23 + 1e-40).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_near_ties(device, score, bias, groups):
    """Scores that differ by less than float32 can say are ordered as float64 orders them."""
    T, E, k = 64, 96, 8
    g = torch.Generator().manual_seed(3)
    x = torch.randn(T, 1, generator=g).expand(T, E).clone()
    for _ in range(3):  # runs of neighbouring float32 values, in random order
        step = torch.randint(0, 2, (T, E), generator=g).bool()
        x = torch.where(step, torch.nextafter(x, torch.tensor(9.0)), x)
    b = (0.5 + torch.randn(E, generator=g) * 1e-7) if bias else None
    w, ids = ops.route_experts(x.to(device), k, score=score, bias=None if b is None else b.to(device),
                               num_groups=groups, top_groups=min(2, groups))
    rw, rids = route_ref(x, k, score, b, groups, min(2, groups), True, 1.0)
    assert torch.equal(ids.cpu(), rids)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_masked_rows(device, score, bias, groups):
    """-inf, the type's lowest value, +inf and NaN among the logits; rows of -inf alone."""
    E, k, inf = 16, 6, float("inf")
    g = torch.Generator().manual_seed(4)
    x = torch.randn(7, E, generator=g)
    x[0] = -inf
    x[1, :13] = -inf  # fewer left than are asked for
    x[2] = torch.finfo(torch.float32).min
    x[3, 5] = torch.finfo(torch.float32).min
    x[4, [2, 9]] = float("nan")
    x[5, 3] = inf
    x[6, 1:] = float("nan")
    b = torch.linspace(0.5, -0.5, E) if bias else None
    w, ids = ops.route_experts(x.to(device), k, score=score, bias=None if b is None else b.to(device),
                               num_groups=groups, top_groups=min(3, groups))
    rw, rids = route_ref(x, k, score, b, groups, min(3, groups), True, 1.0)
    assert torch.equal(ids.cpu(), rids)
    assert ((ids >= 0) & (ids < E)).all() and all(len(set(r)) == k for r in ids.tolist())
    w = w.cpu().double()
    assert torch.equal(torch.isnan(w), torch.isnan(rw))
    ok = ~torch.isnan(rw)
    assert ((w[ok] - rw[ok]).abs() <= rw[ok].abs() * 2.0 ** -23 + 1e-40).all()
    assert (w[0] == 0).all()


def expert_ref(x, gate_up, down, weights, ids, half, fp8):
    """float64 result and its bound (None with fp8: see the module's text)."""
    T, H = x.shape
    E, F = down.shape[0], down.shape[2]
    out, tol = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    unit = 2.0 ** -24
    for t in range(T):
        for j in range(ids.shape[1]):
            e = int(ids[t, j])
            if not 0 <= e < E:
                continue
            xt = x[t]
            gu = gate_up[e] @ xt
            dgu = gate_up[e].abs() @ xt.abs() * (H / 8 + 8) * unit
            (g, u), (dg, du) = gu.view(2, F), dgu.view(2, F)
            a = g * torch.sigmoid(g) * u
            da = 1.01 * (1.1 * dg * u.abs() + g.abs() * du) + a.abs() * (2.0 ** -21 + 1.01 * half) + 2.0 ** -25
            if fp8:
                a8, s = quantise(a[None])
                a = (a8 * expand(s, F, 1))[0]
            w = float(weights[t, j])
            y = down[e] @ a
            out[t] += w * y
            # an expert's result waits for the sum as fp16 times a power of two (but for fp16 results of 16-bit weights,
            # whose bound this does not change): 2^-12 of it, and 2^-39 of its row's largest
            wait = y.abs() * 2.0 ** -12 + y.abs().max() * 2.0 ** -39
            tol[t] += abs(w) * (down[e].abs() @ (da + a.abs() * (F / 8 + 8) * unit) + wait)
    return out, tol + out.abs() * (half * 1.01 + 2.0 ** -20) + 2.0 ** -25


def make(T, E, k, H, F, dtype, fp8, seed, device, skew=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H + 8, generator=g).to(dtype)
    wts = torch.rand(T, k, generator=g)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32)
    if skew:
        ids[:, 0] = E - 1  # every token chose one expert (twice, where it was drawn too)
    if fp8:
        gu = [[weights(g, F, H, 0.2) for _ in range(2)] for _ in range(E)]
        dn = [weights(g, H, F, 0.2) for _ in range(E)]
        args = dict(gate_up=torch.stack([torch.cat([p[0] for p in q]) for q in gu]),
                    gate_up_scale=torch.stack([torch.cat([p[1] for p in q]) for q in gu]),
                    down=torch.stack([p[0] for p in dn]), down_scale=torch.stack([p[1] for p in dn]))
        ref = torch.stack([torch.cat([p[2] for p in q]) for q in gu]), torch.stack([p[2] for p in dn])
        x8, s = quantise(x[:, :H].double())
        xr = x8 * expand(s, H, 1)
    else:
        args = dict(gate_up=(torch.randn(E, 2 * F, H, generator=g) * 0.2).to(dtype),
                    down=(torch.randn(E, H, F, generator=g) * 0.2).to(dtype))
        ref = args["gate_up"].double(), args["down"].double()
        xr = x[:, :H].double()
    args = {n: t.to(device) for n, t in args.items()}
    return x.to(device)[:, :H], args, wts.to(device), ids.to(device), xr, ref


def check(got, x, ref, wts, ids, dtype, fp8):
    out, tol = expert_ref(x, *ref, wts.cpu().double(), ids.cpu(), HALF[dtype], fp8)
    err = (got.cpu().double() - out).abs()
    if not fp8:
        assert (err <= tol).all()
        return
    # An e4m3 rounding within float32 error of a border moves by a step, 2^-3 of the value: about 2^-15 of the
    # gated products do, 2^-10.5 of the result's norm; one of them alone is 2^-3 / sqrt(its row's terms).
    norm = out.norm(dim=1)
    assert (err.norm(dim=1) <= 2.0 ** -5 * norm + 1e-12).all()
    assert err.norm() <= 1.01 * HALF[dtype] * norm.norm() + 2.0 ** -9 * norm.norm() + 1e-12


SHAPES = [(1, 4, 1, 64, 16), (1, 8, 8, 256, 96), (5, 3, 2, 144, 160), (40, 5, 3, 272, 128), (17, 64, 8, 128, 48),
          (150, 4, 2, 128, 272), (300, 2, 2, 160, 144)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,H,F", SHAPES)
def test_expert_mlp(device, T, E, k, H, F, dtype, fp8):
    x, args, wts, ids, xr, ref = make(T, E, k, H, F, dtype, fp8, T + H, device)
    got = ops.expert_mlp(x, weights=wts, ids=ids, **args)
    check(got, xr, ref, wts, ids, dtype, fp8)


@pytest.mark.parametrize("fp8", [False, True])
def test_expert_mlp_ids(device, fp8):
    """One expert for every token and twice in some rows, others that got none; ids
    of another rank (below 0) and of nobody; a row with no expert left."""
    T, E, k, H, F = 90, 6, 3, 128, 80
    x, args, wts, ids, xr, ref = make(T, E, k, H, F, torch.bfloat16, fp8, 3, device, skew=True)
    ids[4] = -1
    ids[7] = torch.tensor([2, 2, 2], dtype=torch.int32)
    ids[8, 1] = -5
    status = ops.new_status(device)
    wide = torch.full((T + 1, H + 8), 3.0, dtype=torch.bfloat16, device=device)
    got = ops.expert_mlp(x, weights=wts, ids=ids, status=status, out=wide[:T, :H], **args)
    ops.check_status(status)
    check(got, xr, ref, wts, ids, torch.bfloat16, fp8)
    assert (got[4] == 0).all() and (wide[T] == 3).all() and (wide[:, H:] == 3).all()
    ids[9, 2] = E
    ids[10, 0] = 2 ** 31 - 1
    got = ops.expert_mlp(x, weights=wts, ids=ids, status=status, **args)
    check(got, xr, ref, wts, ids, torch.bfloat16, fp8)
    with pytest.raises(ValueError, match="expert id"):
        ops.check_status(status)
    ids.fill_(-1)
    assert (ops.expert_mlp(x, weights=wts, ids=ids, **args) == 0).all()
    assert ops.expert_mlp(x[:0], weights=wts[:0], ids=ids[:0], **args).shape == (0, H)


@pytest.mark.parametrize("fp8", [False, True])
def test_expert_mlp_bad_rows_stay_their_own(device, fp8):
    """NaN and infinite rows reach their own results only, also inside a shared tile."""
    T, E, k, H, F = 50, 3, 2, 128, 64
    x, args, wts, ids, xr, ref = make(T, E, k, H, F, torch.bfloat16, fp8, 5, device)
    clean = ops.expert_mlp(x, weights=wts, ids=ids, **args)
    x = x.clone()
    x[11, 3] = float("nan")
    x[30, 7] = float("inf")
    got = ops.expert_mlp(x, weights=wts, ids=ids, **args)
    rest = [i for i in range(T) if i not in (11, 30)]
    assert torch.equal(got[rest], clean[rest])
    assert torch.isnan(got[11]).all() and not torch.isfinite(got[30]).all()


@pytest.mark.parametrize("T", [3, 3000])
def test_expert_mlp_is_the_same_every_time(device, T):
    """Where a row lands among its expert's differs between runs; results do not.
    A workspace full of NaN changes nothing either."""
    E, k, H, F = 7, 4, 128, 64
    x, args, wts, ids, _, _ = make(T, E, k, H, F, torch.bfloat16, True, 6, device)
    first = ops.expert_mlp(x, weights=wts, ids=ids, **args)
    ws = torch.full((ops.expert_mlp_workspace_bytes(T, k, E, H, F, True),), 0xFF, dtype=torch.uint8, device=device)
    for _ in range(3):
        assert torch.equal(ops.expert_mlp(x, weights=wts, ids=ids, workspace=ws, **args), first)
    half = T // 2 + 1  # a token alone, or with others
    assert torch.equal(ops.expert_mlp(x[:half], weights=wts[:half], ids=ids[:half], **args), first[:half])


def test_many_choices_are_sorted(device):
    """More choices than one workgroup sorts, over many experts: each token's result is
    its own experts', told by weights of one expert's number each."""
    T, E, k, H, F = 5000, 600, 4, 16, 16
    g = torch.Generator().manual_seed(8)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32)
    ids[torch.rand(T, k, generator=g) < 0.2] = -1
    x = torch.zeros(T, H)
    x[:, 0] = 1.0
    gu = torch.zeros(E, 2 * F, H)
    gu[:, 0, 0] = 20.0  # silu(20) = 20 to bf16
    gu[:, F, 0] = 1.0
    dn = torch.zeros(E, H, F)
    dn[:, 0, 0] = torch.arange(E) // 256
    dn[:, 1, 0] = torch.arange(E) % 256
    bf = lambda t: t.to(torch.bfloat16).to(device)
    wts = torch.full((T, k), 1.0 / 20)
    got = ops.expert_mlp(bf(x), bf(gu), bf(dn), wts.to(device), ids.to(device)).cpu().double()
    v = ids.double()
    want = torch.where(ids >= 0, v // 256, 0).sum(1), torch.where(ids >= 0, v % 256, 0).sum(1)
    for c in range(2):
        assert ((got[:, c] - want[c]).abs() <= want[c] * (2.0 ** -8 + 1e-6) + 1e-6).all()
    assert (got[:, 2:] == 0).all()


def test_captured_layer(device):
    """Router and experts captured as one graph and replayed on new tokens, with eager calls in between."""
    T, E, k, H, F = 45, 12, 3, 256, 96
    x, args, _, _, _, ref = make(T, E, k, H, F, torch.bfloat16, True, 9, device)
    router = torch.randn(E, H, generator=torch.Generator().manual_seed(1)).to(device)

    def layer(x):
        w, ids = ops.route_experts(x.float() @ router.t(), k, score="sigmoid")
        return ops.expert_mlp(x, weights=w, ids=ids, **args), w, ids

    xs = [torch.randn(T, H, generator=torch.Generator().manual_seed(20 + i)).to(torch.bfloat16).to(device)
          for i in range(3)]
    static = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, w, ids = layer(static)
    for x in xs + xs:
        eager = layer(x)
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((out, w, ids), eager):
            assert torch.equal(a, b)
        x8, s = quantise(x.cpu().double())
        check(out, x8 * expand(s, H, 1), ref, w, ids, torch.bfloat16, True)
