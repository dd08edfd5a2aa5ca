"""GPU tests of `route_experts` and `combine_experts` against the definitions in 64 bits.

Experts, offsets, rows and places are whole numbers and have to be equal.  A weight is computed in 64 bits and rounded once, half a unit of
its last place (2^-24 of it); the softmax that is not renormalized has a sum of up to 1024 terms in 32 bits, 32 a lane and each of them off by a unit of its
last place at the most: 40 * 2^-24.  A combined row is off by a rounding of each of its k products and sums and one to its type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def ops():
    from ac4k_kernel_amd import ops as o
    return o


def reference(logits, k, scoring="softmax", bias=None, groups=1, top_groups=None, group_best=1, renormalize=True, scale=1.0):
    """One token after the other, by the definition."""
    x = logits.detach().cpu().double().reshape(-1, logits.shape[-1])
    t, e = x.shape
    top_groups = groups if top_groups is None else top_groups
    weights, experts = torch.zeros((t, k), dtype=torch.float64), torch.full((t, k), -1)
    for i in range(t):
        if scoring == "softmax":
            p = torch.exp(x[i] - x[i].max())
            score = (p / p.sum()).tolist()
        else:
            score = torch.sigmoid(x[i]).tolist()
        key = list(score) if bias is None else [s + b for s, b in zip(score, bias.cpu().double().tolist())]
        row = x[i].tolist()
        if bias is None and group_best == 1:
            key = row  # the same order, without roundings
        allowed = [j for j in range(e) if row[j] != -math.inf and key[j] != -math.inf]

        def order(v, j):
            return (0, 0.0, j) if math.isnan(v) else (1, -v, j)
        if top_groups < groups:
            size, rank = e // groups, []
            for g in range(groups):
                best = sorted((order(key[j], j) for j in allowed if j // size == g))[:group_best]
                if best:
                    values = [math.nan if kind == 0 else -v for kind, v, _ in best]
                    rank.append(order(sum(values), g))
            kept = {g for *_, g in sorted(rank)[:top_groups]}
            allowed = [j for j in allowed if j // size in kept]
        for s, (*_, j) in enumerate(sorted(order(key[j], j) for j in allowed)[:k]):
            experts[i, s], weights[i, s] = j, score[j]
    if renormalize:
        total = weights.sum(1, keepdim=True)
        weights = torch.where(total == 0, 0.0, weights / total)
    offsets, rows, places = [0], [], torch.full((t, k), -1)
    for j in range(e):
        for i, s in (experts == j).nonzero().tolist():
            places[i, s] = len(rows)
            rows.append(i)
        offsets.append(len(rows))
    rows += [-1] * (t * k - len(rows))
    return weights * scale, experts, torch.tensor(offsets), torch.tensor(rows), places


def check(got, want, rtol=2.0 ** -24):
    lead = got[0].shape
    for g, w, name in zip(got[1:], want[1:], ("experts", "offsets", "rows", "places")):
        assert g.dtype == torch.int32
        assert torch.equal(g.cpu().long().reshape(w.shape), w), name
    w = want[0].reshape(lead)
    g = got[0].cpu().double()
    assert got[0].dtype == torch.float32 and torch.equal(g.isnan(), w.isnan())
    assert bool(((g - w).abs() <= rtol * w.abs() + 2.0 ** -149)[~w.isnan()].all()), (g - w).abs().max()


def logits_of(t, e, dtype="fp32", seed=0, std=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((t, e), generator=g) * std).to(DTYPES[dtype])


def bias_of(e, seed=0, std=0.1):
    return torch.randn((e,), generator=torch.Generator().manual_seed(seed + 99)) * std


SHAPES = [(1, 1, 1), (1, 8, 2), (3, 5, 5), (16, 64, 8), (17, 60, 4), (64, 128, 8), (65, 128, 16), (64, 33, 17), (63, 1000, 64), (130, 256, 8), (129, 97, 6),
          (200, 512, 6), (66, 1024, 8), (257, 16, 2), (1025, 32, 4), (100, 1, 1), (100, 3, 2), (70, 9, 4), (65, 7, 7),
          (128, 64, 16), (192, 128, 4), (255, 17, 3), (256, 100, 8), (300, 1, 1), (300, 3, 2), (290, 9, 4), (270, 7, 7), (129, 64, 17)]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,e,k", SHAPES)
def test_choice_by_logits(t, e, k, scoring):
    x = logits_of(t, e, "bf16", seed=t + e)  # 16 bits: many logits are equal
    for renormalize in (True, False):
        got = ops().route_experts(x.cuda(), k, scoring=scoring, renormalize=renormalize, scale=2.5)
        check(got, reference(x, k, scoring, renormalize=renormalize, scale=2.5), 2.0 ** -24 if renormalize or scoring == "sigmoid" else 40 * 2.0 ** -24)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,e,k", SHAPES)
def test_choice_by_keys_with_a_bias(t, e, k, scoring):
    x, b = logits_of(t, e, "fp16", seed=t + e), bias_of(e)
    got = ops().route_experts(x.cuda(), k, scoring=scoring, bias=b.cuda(), renormalize=e % 2 == 0)
    check(got, reference(x, k, scoring, b, renormalize=e % 2 == 0))


@pytest.mark.parametrize("e,groups,top_groups,k", [(8, 2, 1, 2), (256, 8, 4, 8), (96, 3, 2, 6), (160, 8, 3, 6), (64, 64, 5, 5), (1024, 2, 1, 8), (1020, 5, 2, 9),
                                                   (1023, 33, 7, 8), (100, 10, 10, 4), (48, 16, 1, 3), (12, 4, 2, 6)])
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("biased", [False, True])
def test_groups(e, groups, top_groups, k, best, biased):
    for t in (7, 70):
        x, b = logits_of(t, e, "fp32", seed=e), bias_of(e) if biased else None
        args = dict(scoring="sigmoid" if e % 3 else "softmax", groups=groups, top_groups=top_groups, group_best=best)
        check(ops().route_experts(x.cuda(), k, bias=None if b is None else b.cuda(), **args), reference(x, k, bias=b, **args))


@pytest.mark.parametrize("t", [1, 16, 64, 100])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("e", [64, 300])
def test_equal_keys_go_to_the_lowest_index(t, e, biased):
    x, b = torch.zeros((t, e)), torch.zeros(e) if biased else None
    x[:, 1::2] = -0.0
    x[t // 2:, e // 2:] = 1.0
    got = ops().route_experts(x.cuda(), 5, bias=None if b is None else b.cuda())
    check(got, reference(x, 5, bias=b))
    assert got[1][0].tolist() == ([0, 1, 2, 3, 4] if t > 1 else list(range(e // 2, e // 2 + 5)))


@pytest.mark.parametrize("t", [5, 90])
@pytest.mark.parametrize("groups", [1, 4])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_masked_experts(t, groups, biased, scoring):
    e, k = 64, 6
    x, b = logits_of(t, e), bias_of(e) if biased else None
    x[0] = -math.inf                # a row without experts
    x[1, 3:] = -math.inf            # fewer than k
    x[2, :50] = -math.inf           # groups without experts
    x[3, ::2] = torch.finfo(torch.float32).min
    if biased:
        b[7] = -math.inf            # an expert that nobody takes
        b[9] = math.inf             # and one that everybody does
    args = dict(scoring=scoring, groups=groups, top_groups=min(2, groups), group_best=1 + biased)
    got = ops().route_experts(x.cuda(), k, bias=None if b is None else b.cuda(), **args)
    want = reference(x, k, bias=b, **args)
    check(got, want)
    assert got[1][0].tolist() == [-1] * k and got[0][0].tolist() == [0.0] * k and got[4][0].tolist() == [-1] * k
    assert (got[3][got[2][-1]:] == -1).all()
    if biased:
        assert not (got[1] == 7).any()


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_values_that_are_not_finite(scoring, biased):
    x, b = logits_of(80, 64), bias_of(64) if biased else None
    clean = ops().route_experts(x.cuda(), 4, scoring=scoring, bias=None if b is None else b.cuda())
    x[2, 10], x[70, 60], x[71, 5] = math.nan, math.nan, math.inf
    got = ops().route_experts(x.cuda(), 4, scoring=scoring, bias=None if b is None else b.cuda())
    assert got[0][2].isnan().any() and got[0][70].isnan().any()
    assert got[0][71].isnan().any() == (scoring == "softmax")
    others = [i for i in range(80) if i not in (2, 70, 71)]
    assert torch.equal(got[0][others], clean[0][others]) and torch.equal(got[1][others], clean[1][others])
    assert ((got[1] >= 0) & (got[1] < 64)).all() and got[2][-1] == 320
    if scoring == "sigmoid":
        check(got, reference(x, 4, scoring, b))


def test_large_values_without_a_sum():
    x = torch.full((3, 8), -200.0)  # scores that 32 bits do not have
    x[1], x[2] = 20000.0, -20000.0  # and that 64 do not
    got = ops().route_experts(x.cuda(), 2, scoring="sigmoid")
    check(got, reference(x, 2, "sigmoid"))
    assert got[0].tolist() == [[0.5, 0.5], [0.5, 0.5], [0.0, 0.0]]


@pytest.mark.parametrize("biased", [False, True])
def test_strides_and_leading_dims(biased):
    wide = logits_of(6 * 30, 80).reshape(6, 30, 80).cuda()
    b = bias_of(60).cuda() if biased else None
    for x in (wide[:, :, 7:67], wide[:, :, :60].transpose(0, 1), wide[::2, :, 10:70], wide[:, :, :60].permute(1, 0, 2).contiguous().permute(1, 0, 2), wide[0, 0, :60]):
        got = ops().route_experts(x, 4, bias=b)
        assert got[0].shape == got[1].shape == got[4].shape == (*x.shape[:-1], 4)
        check(got, reference(x.contiguous(), 4, bias=b))


def test_no_tokens():
    for shape in ((0, 16), (3, 0, 16)):
        weights, experts, offsets, rows, places = ops().route_experts(torch.zeros(shape, device="cuda"), 4)
        assert weights.shape == experts.shape == places.shape == (*shape[:-1], 4) and rows.shape == (0,)
        assert offsets.tolist() == [0] * 17
        assert ops().combine_experts(torch.zeros((0, 32), device="cuda"), weights, places).shape == (*shape[:-1], 32)


@pytest.mark.parametrize("t,e,k,biased", [(5000, 128, 4, False), (4001, 256, 8, True), (70000, 64, 2, False), (20000, 1000, 3, True)])
def test_plan_of_many_tokens(t, e, k, biased):
    x = logits_of(t, e, "bf16", seed=3).cuda()
    x[t - t // 20:] = -math.inf
    weights, experts, offsets, rows, places = ops().route_experts(x, k, bias=bias_of(e).cuda() if biased else None)
    top = x.float().sort(dim=1, descending=True, stable=True)
    if not biased:
        met = torch.arange(t, device="cuda")[:, None] < t - t // 20
        assert torch.equal(experts.long(), torch.where(met, top.indices[:, :k], -1))
    flat = torch.where(experts < 0, e, experts).reshape(-1)
    order = flat.sort(stable=True).indices
    count = torch.bincount(flat, minlength=e + 1)[:e]
    total = int(count.sum())
    assert torch.equal(offsets.long(), torch.cat((count.new_zeros(1), count.cumsum(0))))
    assert torch.equal(rows[:total].long(), order[:total] // k) and (rows[total:] == -1).all()
    assert torch.equal(places.reshape(-1)[order[:total]].long(), torch.arange(total, device="cuda"))


def test_a_second_call_and_another_stream_give_the_same():
    x, b = logits_of(3000, 256).cuda(), bias_of(256).cuda()
    first = ops().route_experts(x, 8, bias=b, groups=8, top_groups=4, group_best=2)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(ops().route_experts(x, 8, bias=b, groups=8, top_groups=4, group_best=2))
    torch.cuda.synchronize()
    for other in got:
        assert all(torch.equal(p, q) for p, q in zip(first, other))


@pytest.mark.parametrize("t", [16, 1000])
def test_captured(t):
    x, r = logits_of(t, 64).cuda(), torch.randn((t, 256), device="cuda")
    y = torch.randn((t * 4, 256), device="cuda")
    ops().combine_experts(y, *[ops().route_experts(x, 4)[i] for i in (0, 4)], residual=r)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = ops().route_experts(x, 4)
        out = ops().combine_experts(y, plan[0], plan[4], residual=r)
    for seed in range(4):
        x.copy_(logits_of(t, 64, seed=seed + 5))
        x[seed * 3:seed * 3 + seed] = -math.inf
        graph.replay()
        torch.cuda.synchronize()
        eager = ops().route_experts(x, 4)
        assert all(torch.equal(p, q) for p, q in zip(plan, eager))
        assert torch.equal(out, ops().combine_experts(y, eager[0], eager[4], residual=r))


# ------------------------------------------------------------------------------------------------------------- combine
def combined(y, weights, places, residual=None):
    """(sum, sum of magnitudes) in 64 bits on the CPU."""
    y, w, p = y.cpu().double(), weights.cpu().double(), places.cpu().long()
    lead, k = p.shape[:-1], p.shape[-1]
    w, p = w.reshape(-1, k), p.reshape(-1, k)
    out = torch.zeros((p.shape[0], y.shape[1]), dtype=torch.float64)
    size = torch.zeros_like(out)
    if residual is not None:
        out += residual.cpu().double().reshape(out.shape)
        size += out.abs()
    for s in range(k):
        for i in range(p.shape[0]):
            if 0 <= p[i, s] < y.shape[0]:
                out[i] += w[i, s] * y[p[i, s]]
                size[i] += (w[i, s] * y[p[i, s]]).abs()
    return out.reshape(*lead, -1), size.reshape(*lead, -1)


def close(got, exact, size, k):
    eps = torch.finfo(got.dtype).eps / 2
    least = 2.0 ** -25 if got.dtype == torch.float16 else 0.0  # half a step of fp16 next to zero
    bound = exact.abs() * eps * (1 + eps) + (k + 1) * 2.0 ** -24 * size * 1.01 + least
    diff = (got.cpu().double() - exact).abs()
    assert bool((diff <= bound).all()), (diff - bound).max()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("t,k,n", [(1, 1, 1), (1, 8, 4096), (5, 3, 7), (16, 8, 2049), (33, 2, 5003), (70, 6, 128), (9, 17, 264)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_combine(t, k, n, dtype, with_residual):
    g = torch.Generator().manual_seed(t * k + n)
    y = torch.randn((t * k, n), generator=g).to(DTYPES[dtype])
    places = torch.randperm(t * k, generator=g).reshape(t, k).to(torch.int32)
    places[t // 2, 0] = -1
    places[t - 1, k - 1] = t * k        # behind the last row
    weights = torch.rand((t, k), generator=g)
    r = torch.randn((t, n), generator=g).to(DTYPES[dtype]) if with_residual else None
    got = ops().combine_experts(y.cuda(), weights.cuda(), places.cuda(), residual=None if r is None else r.cuda())
    assert got.dtype == DTYPES[dtype] and got.shape == (t, n)
    close(got, *combined(y, weights, places, r), k)


def test_combine_of_no_place_is_the_residual():
    r = torch.randn((4, 100), device="cuda")
    y = torch.full((8, 100), math.nan, device="cuda")
    places = torch.full((4, 2), -1, dtype=torch.int32, device="cuda")
    assert torch.equal(ops().combine_experts(y, torch.full((4, 2), math.nan, device="cuda"), places, residual=r), r)
    assert (ops().combine_experts(y, torch.ones((4, 2), device="cuda"), places) == 0).all()
    assert (ops().combine_experts(y[:0], torch.ones((4, 2), device="cuda"), torch.zeros_like(places)) == 0).all()


def test_combine_into_the_residual_and_strided_operands():
    g = torch.Generator().manual_seed(2)
    wide = torch.randn((24, 300), generator=g).to(torch.bfloat16).cuda()
    y, k = wide[:, 3:203], 3
    places = torch.arange(24, dtype=torch.int32).reshape(2, 4, 3).cuda()
    weights = torch.rand((2, 4, 3), generator=g).cuda()
    buffer = torch.randn((8, 256), generator=g).to(torch.bfloat16).cuda()
    r = buffer[:, 5:205].unflatten(0, (2, 4))
    exact = combined(y, weights, places, r)
    before = buffer.clone()
    out = ops().combine_experts(y, weights, places, residual=r)
    close(out, *exact, k)
    got = ops().combine_experts(y, weights, places, residual=r, out=r)
    assert got is r and torch.equal(r, out)
    assert torch.equal(buffer[:, :5], before[:, :5]) and torch.equal(buffer[:, 205:], before[:, 205:])
    # columns apart: copied
    assert torch.equal(ops().combine_experts(y.t().contiguous().t(), weights, places, residual=before[:, 5:205].t().contiguous().t().unflatten(0, (2, 4))), out)


def test_combine_on_rows_that_are_read_often():
    y = torch.randn((7, 520), device="cuda", dtype=torch.float16)
    places = torch.zeros((50, 4), dtype=torch.int32, device="cuda")
    places[:, 2] = 6
    weights = torch.full((50, 4), 0.25, device="cuda")
    r = torch.randn((1, 520), device="cuda", dtype=torch.float16).expand(50, 520)
    got = ops().combine_experts(y, weights, places, residual=r)
    close(got, *combined(y, weights, places, r), 4)
    assert (got == got[0]).all()


def test_routing_of_an_output_that_records_gradients():
    x = torch.randn((20, 32), device="cuda", requires_grad=True)
    got = ops().route_experts(x * 2, 3)
    check(got, reference(x * 2, 3))
    assert not any(t.requires_grad for t in got)


def test_python_refusals_of_combine():
    y, w, p = torch.zeros((8, 64), device="cuda"), torch.zeros((4, 2), device="cuda"), torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    r = torch.zeros((4, 64), device="cuda")
    c = ops().combine_experts
    for kw in (dict(y=y.cpu()), dict(y=y[0]), dict(y=y.double()), dict(weights=w.half()), dict(weights=w[:3]), dict(weights=w.t()), dict(places=p.long()), dict(places=p[:, :0], weights=w[:, :0]),
               dict(residual=r.half()), dict(residual=r[:3]), dict(residual=r[:, :32]), dict(residual=1.0), dict(out=r.half()), dict(out=r[:2]), dict(out=y[:4]),
               dict(out=r[0].expand(4, 64)), dict(residual=y.flatten()[:256].view(4, 64), out=y.flatten()[64:320].view(4, 64)), dict(places=[0]), dict(weights=1.0), dict(out=2)):
        with pytest.raises(RuntimeError):
            c(**{**dict(y=y, weights=w, places=p), **kw})


def test_python_refusals_of_route():
    x = torch.zeros((4, 64), device="cuda")
    r = ops().route_experts
    for kw in (dict(logits=x.cpu()), dict(logits=x.double()), dict(logits=[1.0]), dict(logits=x[:, :0]), dict(top_k=0), dict(top_k=65), dict(top_k=2.0), dict(top_k=None), dict(groups="2"), dict(logits=x[:, :4], top_k=5), dict(scoring="relu"),
               dict(bias=torch.zeros(63, device="cuda")), dict(bias=torch.zeros(64)), dict(bias=torch.zeros(64, device="cuda").half()), dict(bias=0.0), dict(groups=3),
               dict(groups=0), dict(groups=4, top_groups=5), dict(groups=4, top_groups=0), dict(groups=4, top_groups=1, top_k=17), dict(group_best=3),
               dict(logits=torch.zeros((2, 1025), device="cuda"))):
        with pytest.raises(RuntimeError):
            r(**{**dict(logits=x, top_k=2), **kw})
