"""The MoE layer and router for a few tokens against plain formulas in 64 bits.

Tolerances follow the roundings: hidden to bf16 (2^-8 of each value at most) between the products, the output to bf16 (2^-8), and
fp32 sums, off by 2^-23 of the sum of magnitudes for every addition that a term passes through (16 within an mma, one per mma of its
warp, 8 for the warps); each is carried through the products that follow it.  That bounds every element for the worst signs.  The
errors' signs are as random as the inputs here, so their norm over all outputs is also held to 2^-7 of the result's: 2^-8 for
the rounding of hidden and 2^-8 for that of the output."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -8


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import mok  # noqa: F401
    return torch.device("cuda", 0)


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _normal(dev, *shape, std=1.0, seed=0, dtype=torch.bfloat16):
    return torch.empty(shape, device=dev, dtype=torch.float32).normal_(0.0, std, generator=_gen(dev, seed)).to(dtype)


def _layer(dev, T, H, I, E, K, *, shared=0, fp8=False, total=None, seed=0):
    """x, routes, weights, shared weights, routed weights (bf16, or codes and scales of any fp32 value)."""
    x = _normal(dev, T, H, seed=seed)
    scores = torch.rand(T, total or E, device=dev, generator=_gen(dev, seed + 1))
    w, routes = torch.topk(scores, K, dim=1)
    weights = torch.softmax(4 * w, dim=1)
    shapes = ((E, I, H), (E, I, H), (E, H, I))
    if fp8:
        routed = tuple((_normal(dev, *s, std=100.0, seed=seed + 2 + i, dtype=torch.float32).clamp_(-448, 448).to(torch.float8_e4m3fn),
                        torch.rand(s[0], -(-s[1] // 128), -(-s[2] // 128), device=dev, generator=_gen(dev, seed + 5 + i))
                        .add_(0.5).mul_(0.01 * s[2] ** -0.5)) for i, s in enumerate(shapes))
    else:
        routed = tuple(_normal(dev, *s, std=s[2] ** -0.5, seed=seed + 2 + i) for i, s in enumerate(shapes))
    sh = (None,) * 3
    if shared:
        sh = tuple(_normal(dev, *s, std=s[1] ** -0.5, seed=seed + 8 + i) for i, s in enumerate(((shared, H), (shared, H), (H, shared))))
    return x, routes.to(torch.int32), weights, sh, routed


def _dense(w, e):
    if not isinstance(w, tuple):
        return w[e].double()
    q, s = w[0][e], w[1][e].double()
    return q.double() * s.repeat_interleave(128, 0)[: q.shape[0]].repeat_interleave(128, 1)[:, : q.shape[1]]


def _additions(n):
    return 24 + 2 * -(-n // 256)


def _expert(x, g, u, d, limit):
    """Output, its bound from the roundings before the last, and the sum of magnitudes of its last product."""
    gate, up = x @ g.t(), x @ u.t()
    d_gate, d_up = [_additions(x.shape[1]) * 2.0 ** -23 * (x.abs() @ w.abs().t()) for w in (g, u)]
    if limit is not None:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
    silu = gate * torch.sigmoid(gate)
    h = silu * up
    d_h = (BF16 + 2.0 ** -19) * 1.01 * h.abs() + 1.1 * d_gate * (up.abs() + d_up) + silu.abs() * d_up
    return h @ d.t(), d_h @ d.abs().t(), h.abs() @ d.abs().t()


def _reference(x, routes, weights, shared, routed, first=0, limit=None):
    x, weights = x.double(), weights.double()
    E, I = (routed[0][0] if isinstance(routed[0], tuple) else routed[0]).shape[:2]
    out, tol, size = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    terms = _additions(I) + routes.shape[1] + 1
    if shared[0] is not None:
        parts = _expert(x, *(w.double() for w in shared), limit)
        for t, p in zip((out, tol, size), parts):
            t += p
        terms = max(terms, _additions(shared[0].shape[0]) + routes.shape[1] + 1)
    for e in range(E):
        t, k = torch.nonzero(routes == first + e, as_tuple=True)
        if t.numel():
            parts = _expert(x[t], *(_dense(w, e) for w in routed), limit)
            w = weights[t, k][:, None]
            for acc, p, f in zip((out, tol, size), parts, (w, w.abs(), w.abs())):
                acc.index_add_(0, t, f * p)
    return out, tol * 1.01 + BF16 * 1.01 * out.abs() + terms * 2.0 ** -23 * size


def _check(dev, args, **kw):
    import mok
    x, routes, weights, shared, routed = args
    got = mok.moe_decode(x, routes, weights, *shared, *routed, **{{"first": "first_expert", "limit": "swiglu_limit"}[k]: v for k, v in kw.items()})
    torch.cuda.synchronize()
    mok.ops.check_status(dev)
    want, tol = _reference(*args, **kw)
    off = (got.double() - want).abs()
    assert got.shape == x.shape and bool((off <= tol).all()), f"{(off / tol.clamp_min(1e-30)).max().item():.3f} of the bound"
    assert off.norm() <= 2.0 ** -7 * want.norm()
    return got


CASES = [
    # T, H, I, E, K, shared
    (1, 64, 64, 1, 1, 0), (1, 2048, 768, 128, 8, 768), (2, 128, 192, 4, 2, 64), (3, 320, 128, 7, 3, 0), (7, 1024, 448, 8, 2, 448),
    (8, 512, 256, 16, 4, 256), (9, 512, 256, 16, 4, 320), (16, 7168, 128, 6, 2, 0), (17, 256, 2048, 5, 5, 64), (31, 576, 320, 60, 6, 128),
    (32, 2048, 768, 16, 8, 768), (33, 192, 64, 3, 1, 64), (64, 640, 384, 40, 8, 0), (100, 448, 192, 9, 2, 192), (255, 256, 128, 12, 3, 64),
    (256, 1024, 128, 128, 16, 64), (128, 64, 64, 1024, 32, 0), (5, 16384, 64, 2, 1, 64),
    (7, 64, 64, 1024, 32, 64), (9, 16384, 64, 2, 1, 64),
]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T,H,I,E,K,shared", CASES)
def test_layer(dev, T, H, I, E, K, shared, fp8):
    args = _layer(dev, T, H, I, E, K, shared=shared, fp8=fp8)
    got = _check(dev, args)
    assert torch.equal(got, _check(dev, args))      # no order left to chance


@pytest.mark.parametrize("fp8", [False, True])
def test_clamped(dev, fp8):
    args = _layer(dev, 6, 256, 128, 4, 2, shared=128, fp8=fp8)
    free = _check(dev, args)
    assert not torch.equal(free, _check(dev, args, limit=0.5))
    _check(dev, args, limit=0)


@pytest.mark.parametrize("T", [1, 12, 80, 256])
def test_one_expert_takes_every_token(dev, T):
    args = list(_layer(dev, T, 256, 192, 5, 1, shared=64))
    args[1] = torch.full_like(args[1], 3)
    _check(dev, args)


def test_routes_to_other_ranks_and_to_nobody(dev):
    import mok
    x, routes, weights, shared, routed = _layer(dev, 21, 256, 128, 4, 6, shared=64, total=16)
    for first in (0, 5, 12):
        _check(dev, (x, routes, weights, shared, routed), first=first)
        _check(dev, (x, routes, weights, (None,) * 3, routed), first=first)
    for nobody in (-1, 16, 2 ** 31 - 1, -2 ** 31):
        r = routes.clone()
        r[3], r[7, 2] = nobody, nobody
        got = _check(dev, (x, r, weights, (None,) * 3, routed), first=4)
        assert bool((got[3] == 0).all())
        alone = torch.full_like(r, nobody)
        assert bool((mok.moe_decode(x, alone, weights, None, None, None, *routed) == 0).all())
        _check(dev, (x, alone, weights, shared, routed))
    wide = routes.long()
    wide[0, 0], wide[1, 1], wide[2, 2] = 2 ** 32 + 5, -2 ** 40, 2 ** 31
    narrow = torch.where((wide < 0) | (wide >= 16), -1, wide).to(torch.int32)
    a, b = (mok.moe_decode(x, r, weights, *shared, *routed, first_expert=4) for r in (wide, narrow))
    assert torch.equal(a, b)


def test_an_expert_named_twice(dev):
    args = list(_layer(dev, 40, 128, 64, 3, 8, shared=0, total=8))
    args[1] = (torch.arange(320, device=dev, dtype=torch.int32).reshape(40, 8) * 7 % 5) % 4
    _check(dev, args)
    args[1] = torch.zeros_like(args[1])
    _check(dev, args)


def test_weights_as_they_come(dev):
    """Negative, zero, large and non-finite router weights."""
    import mok
    x, routes, weights, shared, routed = _layer(dev, 10, 128, 64, 6, 3)
    weights = weights * torch.tensor([-3.0, 0.0, 1e4], device=dev)
    _check(dev, (x, routes, weights, shared, routed))
    clean = mok.moe_decode(x, routes, weights, *shared, *routed)
    weights[4, 1], x[6, 17] = float("nan"), float("inf")
    got = mok.moe_decode(x, routes, weights, *shared, *routed)
    assert bool(got[4].isnan().all()) and not bool(got[6].isfinite().any())
    keep = [t for t in range(10) if t not in (4, 6)]
    assert torch.equal(got[keep], clean[keep])      # other tokens are not touched
    gate = routed[0].clone()
    gate[int(routes[2, 0]), 5, 9] = float("nan")
    got = mok.moe_decode(x, routes, weights, *shared, gate, *routed[1:], swiglu_limit=1.0)
    hit = (routes == routes[2, 0]).any(1)
    assert bool(got[hit].isnan().any(1).all()) and torch.equal(got[~hit].isnan().any(1), torch.tensor([t in (4, 6) for t in range(10)], device=dev)[~hit])


def test_every_code(dev):
    """All 256 e4m3 codes, the subnormal ones and NaN included, as weights of the down projection and of the gate."""
    import mok
    H, I = 256, 64
    x = _normal(dev, 3, H)
    codes = torch.arange(256, device=dev, dtype=torch.uint8)
    for e, fill in enumerate((0, 1)):
        down = codes[:, None].expand(H, I).contiguous().view(torch.float8_e4m3fn)[None]
        gate, up = (_normal(dev, 1, I, H, std=40.0, seed=s).to(torch.float8_e4m3fn) for s in (1, 2))
        scale = lambda r, c, v: torch.full((1, -(-r // 128), -(-c // 128)), v, device=dev)  # noqa: E731
        args = [x, torch.zeros(3, 1, device=dev, dtype=torch.int32), torch.ones(3, 1, device=dev), (None,) * 3,
                ((gate, scale(I, H, 0.001)), (up, scale(I, H, 0.001)), (down, scale(H, I, 3.0)))]
        if fill:
            args[4] = ((codes.roll(64 * e)[None, None, :].expand(1, I, H).contiguous().view(torch.float8_e4m3fn), scale(I, H, 1e-4)),) + args[4][1:]
            got = mok.moe_decode(args[0], args[1], args[2], *args[3], *args[4])
            assert bool(got.isnan().all())          # codes 0x7F and 0xFF stand in every row of the gate
            continue
        got = mok.moe_decode(args[0], args[1], args[2], *args[3], *args[4])
        bad = torch.zeros(H, dtype=torch.bool, device=dev)
        bad[0x7F] = bad[0xFF] = True
        assert torch.equal(got.isnan(), bad.expand(3, H))
        clean = down.clone()
        clean.view(torch.uint8)[0, bad] = 0
        args[4] = args[4][:2] + ((clean, args[4][2][1]),)
        want = _check(dev, args)
        assert torch.equal(got[:, ~bad], want[:, ~bad])


def test_a_token_does_not_depend_on_its_batch(dev):
    import mok
    for fp8 in (False, True):
        x, routes, weights, shared, routed = _layer(dev, 256, 256, 192, 6, 2, shared=128, fp8=fp8)
        whole = mok.moe_decode(x, routes, weights, *shared, *routed)
        for part in (slice(0, 1), slice(3, 8), slice(20, 36), slice(30, 94), slice(40, 168), slice(100, 256)):
            assert torch.equal(mok.moe_decode(x[part], routes[part], weights[part], *shared, *routed), whole[part])
        order = torch.randperm(256, device=dev, generator=_gen(dev, 3))
        assert torch.equal(mok.moe_decode(x[order], routes[order], weights[order], *shared, *routed), whole[order])
    w = _normal(dev, 40, 512, std=0.05, dtype=torch.float32)
    y = _normal(dev, 70, 512)
    whole = mok.route_decode(y, w, topk=5)
    for part in (slice(0, 1), slice(3, 8), slice(20, 70)):
        assert all(torch.equal(a, b[part]) for a, b in zip(mok.route_decode(y[part], w, topk=5), whole))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("H,I", [(4672, 2368), (2112, 5184), (576, 64)])
def test_long_sums_do_not_depend_on_the_batch(dev, H, I, fp8):
    """More chunks of the summed dimension than are kept apart, and ragged last ones: few tokens, tiles of few and of many tokens and
    experts of more than one pass all add in one order."""
    import mok
    x, routes, weights, shared, routed = _layer(dev, 150, H, I, 3, 2, shared=128, fp8=fp8)
    whole = _check(dev, (x, routes, weights, shared, routed))
    for part in (slice(0, 1), slice(2, 9), slice(9, 17), slice(20, 52), slice(60, 150)):
        assert torch.equal(mok.moe_decode(x[part], routes[part], weights[part], *shared, *routed), whole[part])


@pytest.mark.parametrize("T", [7, 8, 256])
def test_eight_bit_expert_takes_every_token(dev, T):
    args = list(_layer(dev, T, 320, 192, 70, 2, shared=64, fp8=True))
    args[1] = torch.full_like(args[1], 69)          # named twice by every token
    args[1][0], args[1][T // 2, 1] = 3, 68
    _check(dev, args)
    _check(dev, args[:3] + [(None,) * 3] + args[4:], first=60)


def test_expert_parallel_parts_add_up(dev):
    import mok
    x, routes, weights, shared, routed = _layer(dev, 30, 256, 128, 12, 4, shared=64)
    whole, tol = _reference(x, routes, weights, shared, routed)
    parts = [mok.moe_decode(x, routes, weights, *(shared if r == 0 else (None,) * 3), *(w[4 * r: 4 * r + 4].contiguous() for w in routed),
                            first_expert=4 * r).double() for r in range(3)]
    assert bool(((sum(parts) - whole).abs() <= tol + BF16 * sum(p.abs() for p in parts)).all())


def test_same_as_the_layer(dev, dist_ctx):
    """512 tokens through mok.moe_layer, the same in two calls of 256 here: both are within the layer's own tolerance."""
    import mok
    x, routes, weights, shared, routed = _layer(dev, 512, 256, 256, 8, 2, shared=256)
    layer = mok.moe_layer(x, routes, weights, *shared, *routed)
    few = torch.cat([mok.moe_decode(x[i:i + 256], routes[i:i + 256], weights[i:i + 256], *shared, *routed) for i in (0, 256)])
    off = (layer.double() - few.double()).norm() / few.double().norm()
    assert off <= 1e-2          # two bf16 computations: gate, up, hidden, expert rows and output rounded, 2^-8 at most each


@pytest.mark.parametrize("T", [2, 9])
def test_weights_beyond_31_bits(dev, T):
    H, I, E = 7168, 2048, 160
    args = list(_layer(dev, T, H, 64, 2, 2, shared=0))
    last = _layer(dev, 1, H, I, 2, 2, seed=3)[4]
    routed = []
    for w in last:
        big = torch.empty((E,) + tuple(w.shape[1:]), device=dev, dtype=w.dtype)
        big[-2:] = w
        routed.append(big)
    small, args[4] = (args[0], args[1], args[2], args[3], last), tuple(routed)
    import mok
    got = mok.moe_decode(args[0], args[1] + E - 2, args[2], *args[3], *args[4])
    assert torch.equal(got, _check(dev, small))


def test_strides_and_streams_and_graphs(dev):
    import mok
    x, routes, weights, shared, routed = _layer(dev, 12, 512, 128, 6, 2, shared=64)
    want = mok.moe_decode(x, routes, weights, *shared, *routed)
    wide = torch.full((24, 640), float("nan"), device=dev, dtype=torch.bfloat16)
    view = wide[::2, 64:576]
    view.copy_(x)
    assert torch.equal(mok.moe_decode(view, routes.t().contiguous().t(), weights.t().contiguous().t(), *shared, *routed), want)
    odd = wide[:12, 3:515]
    odd.copy_(x)
    assert torch.equal(mok.moe_decode(odd, routes.long(), weights, *shared, *routed), want)
    # two streams at once
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for rounds in range(10):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(mok.moe_decode(x, routes, weights, *shared, *routed))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(o, want) for o in outs)
    # captured: two graphs with their own inputs, replayed in turn and on two streams
    w_router = _normal(dev, 6, 512, std=0.05, dtype=torch.float32)

    def step(x):
        r, w = mok.route_decode(x, w_router, topk=2)
        return mok.moe_decode(x, r, w, *shared, *routed)
    graphs = []
    for i in range(2):
        xi = x.clone()
        step(xi)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(xi)
        graphs.append((g, xi, out))
    new = [_normal(dev, 12, 512, seed=50 + i) for i in range(2)]
    expect = [step(n) for n in new]
    torch.cuda.synchronize()
    for (g, xi, _), n, s in zip(graphs, new, streams):
        with torch.cuda.stream(s):
            xi.copy_(n)
            for _ in range(20):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, e) for (_, _, out), e in zip(graphs, expect))


@pytest.mark.parametrize("T", [4, 40])
def test_status_word_makes_the_output_nan(dev, T):
    import mok
    args = _layer(dev, T, 128, 64, 2, 1)
    from mok._native import status_word
    status_word(dev).fill_(1)
    try:
        assert bool(mok.moe_decode(args[0], args[1], args[2], *args[3], *args[4]).isnan().all())
    finally:
        status_word(dev).zero_()
    _check(dev, args)


def test_empty_batch(dev):
    import mok
    x, routes, weights, shared, routed = _layer(dev, 2, 128, 64, 2, 1)
    assert mok.moe_decode(x[:0], routes[:0], weights[:0], *shared, *routed).shape == (0, 128)
    r, w = mok.route_decode(x[:0], _normal(dev, 4, 128, dtype=torch.float32), topk=2)
    assert r.shape == w.shape == (0, 2)


# ---- router ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,H,E,K,dtype,bias", [
    (1, 2048, 128, 8, torch.float32, False), (1, 8, 1, 1, torch.float32, True), (3, 264, 5, 5, torch.bfloat16, True),
    (8, 7168, 256, 8, torch.float32, True), (9, 1000, 33, 4, torch.float32, False), (64, 4096, 8, 2, torch.bfloat16, False),
    (256, 512, 1024, 32, torch.float32, True), (255, 2056, 60, 6, torch.float32, False)])
def test_router(dev, T, H, E, K, dtype, bias):
    import mok
    x, w = _normal(dev, T, H), _normal(dev, E, H, std=H ** -0.5, seed=1, dtype=torch.float32).to(dtype)
    b = _normal(dev, E, std=0.5, seed=2, dtype=torch.float32) if bias else None
    routes, weights = mok.route_decode(x, w, b, topk=K)
    logits = x.double() @ w.double().t() + (b.double() if bias else 0.0)
    # fp32 sums: a thread adds at most 8 ceil(H / 2048) products, 13 more additions follow, and the bias
    noise = (8 * -(-H // 2048) + 14) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t()).max() + 2.0 ** -23 * logits.abs().max()
    got = torch.gather(logits, 1, routes.long())
    best = torch.topk(logits, K, dim=1).values
    assert bool((best - got <= 2 * noise).all())                                # the k-th choice is as good as the k-th best
    assert all(len(set(r)) == K for r in routes.tolist())
    want = torch.softmax(got, dim=1)
    assert bool(((weights.double() - want).abs() <= want * (4 * noise + 2.0 ** -20)).all())


def test_router_ties_go_to_the_lower_index(dev):
    import mok
    x = _normal(dev, 5, 64)
    w = _normal(dev, 3, 64, dtype=torch.float32).repeat(4, 1)                   # experts e, e + 3, e + 6, e + 9 are alike
    routes, weights = mok.route_decode(x, w, topk=4)
    best = (x.double() @ w[:3].double().t()).argmax(1)
    assert torch.equal(routes.long(), best[:, None] + 3 * torch.arange(4, device=dev))
    assert bool(((weights - 0.25).abs() < 1e-6).all())


@pytest.mark.parametrize("T", [1, 5, 40, 512])
def test_router_not_finite(dev, T):
    """A token of NaNs chooses experts that there are and its output is NaN, without a shared expert too; experts masked with -inf are
    chosen last, each once, with weight 0.  512: `mok.route`, the same kernel behind another product."""
    import mok
    E, K = 10, 4
    x, w = _normal(dev, T, 256), _normal(dev, E, 256, std=0.05, seed=1, dtype=torch.float32)
    x[T // 2] = float("nan")
    route = mok.route if T == 512 else mok.route_decode
    routes, weights = (t.detach() for t in route(x, w, topk=K))
    assert bool(((routes >= 0) & (routes < E)).all()) and all(len(set(r)) == K for r in routes.tolist())
    assert routes[T // 2].tolist() == [0, 1, 2, 3]                              # alike: the lower index
    bad = torch.zeros(T, dtype=torch.bool, device=dev)
    bad[T // 2] = True
    assert torch.equal(weights.isnan().any(1), bad) and torch.equal(weights.isnan().all(1), bad)
    if T <= 256:
        _, _, _, shared, routed = _layer(dev, T, 256, 64, E, K)
        out = mok.moe_decode(x, routes, weights, *shared, *routed)
        assert torch.equal(out.isnan().all(1), bad) and torch.equal(out.isnan().any(1), bad)
    bias = torch.full((E,), -float("inf"), device=dev)
    bias[[7, 2]] = 0.5
    x[T // 2] = 1.0
    routes, weights = (t.detach() for t in route(x, w, bias, topk=K))
    assert torch.equal(routes[:, :2].sort(1).values, torch.tensor([[2, 7]], dtype=torch.int32, device=dev).expand(T, 2))
    assert torch.equal(routes[:, 2:], torch.tensor([[0, 1]], dtype=torch.int32, device=dev).expand(T, 2))
    # the last one's sum of two exponentials and its division: a few units of 2^-23
    assert bool((weights[:, 2:] == 0).all()) and bool(((weights.sum(1) - 1.0).abs() <= 8 * 2.0 ** -23).all())


def test_router_nan_in_the_matrix(dev):
    """An expert whose logit is NaN comes first, as in torch.topk, and the token's weights are NaN."""
    import mok
    x, w = _normal(dev, 6, 256), _normal(dev, 70, 256, std=0.05, seed=1, dtype=torch.float32)
    w[41] = float("nan")
    routes, weights = mok.route_decode(x, w, topk=3)
    logits = x.double() @ w.double().t()
    assert torch.equal(routes[:, 0], torch.full((6,), 41, dtype=torch.int32, device=dev)) and bool(weights.isnan().all())
    logits[:, 41] = -float("inf")
    best = torch.topk(logits, 2, dim=1)
    gap = (torch.topk(logits, 3, dim=1).values.diff(dim=1).abs().min() > 1e-5).item()
    assert not gap or torch.equal(routes[:, 1:].long(), best.indices)


# ---- as a model uses them ---------------------------------------------------------------------------------------------
def test_serving_step(dev):
    """norm -> router -> experts in 8 bits, and the shared part as 8-bit products, as one captured step with a residual stream."""
    import mok
    T, H, I, E, K = 5, 512, 256, 8, 2
    x, r = _normal(dev, T, H), _normal(dev, T, H, seed=1)
    norm, w_router = _normal(dev, H, seed=2), _normal(dev, E, H, std=0.05, seed=3, dtype=torch.float32)
    full = tuple(_normal(dev, *s, std=s[2] ** -0.5, seed=4 + i) for i, s in enumerate(((E, I, H), (E, I, H), (E, H, I))))
    routed = tuple(mok.quantize_blocks(w, tile_rows=128) for w in full)
    head = mok.quantize_weight(_normal(dev, 1024, H, std=0.05, seed=9), transpose=False)[0]

    def step(x, r):
        y, r = mok.rms_norm(x, norm, r)
        routes, weights = mok.route_decode(y, w_router, topk=K)
        out = mok.moe_decode(y, routes, weights, None, None, None, *routed)
        q, r = mok.rms_norm_quantized(out, norm, r)
        return mok.block_matmul(q, head), r, routes, weights, y, out
    logits, stream, routes, weights, y, out = step(x, r)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        again = step(x, r)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, (logits, stream, routes, weights, y, out)))
    want, tol = _reference(y, routes, weights, (None,) * 3, routed)
    assert bool(((out.double() - want).abs() <= tol).all())
    z = x.double() + r.double()
    assert bool(((stream.double() - (z.bfloat16().double() + out.double())).abs() <= BF16 * stream.double().abs() * 1.01).all())


def test_module(dev, dist_ctx):
    import mok
    torch.manual_seed(0)
    layer = mok.MoKMoE(512, 256, 8, 2, device=dev, swiglu_limit=7.0)
    x = _normal(dev, 512, 512)
    whole = layer(x)
    few = layer.decode(x[:40])
    off = (few.double() - whole[:40].double()).norm() / whole[:40].double().norm()
    assert off <= 1e-2 and not few.requires_grad
    low = layer.decode(x[:40], fp8=True)
    # e4m3 weights: each off by 2^-4 at most; on average over the products' terms well below that
    assert (low.double() - few.double()).norm() / few.double().norm() <= 3 * 2.0 ** -4
    kept = layer._quantized_blocks
    layer.decode(x[:3], fp8=True)
    assert layer._quantized_blocks is kept
    with torch.no_grad():
        layer.w_routed_down.mul_(2.0)
    twice = layer.decode(x[:40], fp8=True)
    assert layer._quantized_blocks is not kept and not torch.equal(twice, low)
    layer.invalidate_quantized()
    assert layer._quantized_blocks is None


def _tuples(copies):
    return [t for pair in copies for t in pair]


def test_module_copies_across_streams(dev, dist_ctx):
    """Copies made on one stream, behind other work of it, are there for a call on another."""
    import mok
    torch.manual_seed(1)
    layer = mok.MoKMoE(512, 256, 8, 2, device=dev)
    x = _normal(dev, 5, 512)
    layer.decode(x, fp8=True)
    first, second = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
    with torch.no_grad():
        for _ in range(3):
            layer.w_routed_up.mul_(-1.5)
            torch.cuda.synchronize()
            with torch.cuda.stream(first):
                torch.cuda._sleep(20_000_000)   # 10 ms
                layer.decode(x, fp8=True)
            with torch.cuda.stream(second):
                got = layer.decode(x, fp8=True)
            torch.cuda.synchronize()
            layer.invalidate_quantized()
            assert torch.equal(got, layer.decode(x, fp8=True))


def test_module_captured_with_copies(dev, dist_ctx):
    """A captured step reads the module's copies: still there, and up to date, after the weights changed and memory was reused."""
    import mok
    torch.manual_seed(2)
    layer = mok.MoKMoE(512, 256, 8, 2, device=dev)
    x = _normal(dev, 5, 512)
    layer.decode(x, fp8=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = layer.decode(x, fp8=True)
    places = [t.data_ptr() for t in _tuples(layer._quantized_blocks[1])]
    for change in (1.0, -3.0, 0.5):
        with torch.no_grad():
            layer.w_routed_gate.mul_(change)
            layer.w_routed_down.mul_(change)
        want = layer.decode(x, fp8=True)
        waste = [torch.full_like(t.view(torch.uint8), 0x7E) for t in _tuples(layer._quantized_blocks[1])]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and [t.data_ptr() for t in _tuples(layer._quantized_blocks[1])] == places
        del waste


def test_module_captured_without_copies(dev, dist_ctx):
    """The first 8-bit call is captured: an eager call before the replay makes its own copies, and the replay gives the same."""
    import mok
    torch.manual_seed(3)
    layer, x = mok.MoKMoE(512, 256, 8, 2, device=dev), _normal(dev, 5, 512)
    layer.decode(x)
    mok.quantize_blocks(layer.w_routed_up.detach(), tile_rows=128)
    other = mok.MoKMoE(512, 256, 8, 2, device=dev)
    other.decode(x, fp8=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = layer.decode(x, fp8=True)
    want = layer.decode(x, fp8=True)
    assert bool(want.isfinite().all()) and layer._quantized_blocks is not None
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    with torch.no_grad():
        layer.w_routed_up.mul_(2.0)
    g.replay()   # quantizes for itself
    torch.cuda.synchronize()
    assert torch.equal(out, layer.decode(x, fp8=True))


def test_traced_calls_match(dev):
    import mok
    x, routes, weights, shared, routed = _layer(dev, 6, 256, 128, 4, 2, shared=64)
    w_router = _normal(dev, 4, 256, std=0.05, dtype=torch.float32)

    @torch.compile(fullgraph=True, backend="aot_eager")
    def f(x):
        r, w = mok.route_decode(x, w_router, topk=2)
        return mok.moe_decode(x, r, w, *shared, *routed, swiglu_limit=2.0), r
    got = f(x)
    r, w = mok.route_decode(x, w_router, topk=2)
    assert torch.equal(got[0], mok.moe_decode(x, r, w, *shared, *routed, swiglu_limit=2.0)) and torch.equal(got[1], r)


def test_gradients_are_not_lost_silently(dev):
    """Inputs that require gradients give outputs whose backward raises, and the same values as without; tangents are refused."""
    import mok
    from torch.autograd import forward_ad
    x, routes, weights, shared, routed = _layer(dev, 6, 256, 128, 4, 2, shared=64)
    w_router, norm = _normal(dev, 4, 256, std=0.05, dtype=torch.float32), _normal(dev, 256)
    a, b = mok.quantize_blocks(x), mok.quantize_blocks(routed[0][0], tile_rows=128)
    calls = [
        (lambda x, w: mok.moe_decode(x, routes, w, *shared, *routed), (x, weights)),
        (lambda x, w: mok.moe_decode(x, routes, weights, *shared, routed[0], w, routed[2]), (x, routed[1])),
        (lambda x, w: mok.route_decode(x, w, topk=2)[1], (x, w_router)),
        (lambda x, w: mok.rms_norm_quantized(x, w, x)[1], (x, norm)),
        (lambda s, t: mok.block_matmul((a[0], s), (b[0], t)), (a[1], b[1])),
    ]
    for call, inputs in calls:
        want = call(*inputs)
        for which in (0, 1):
            leaves = [t.detach().clone(memory_format=torch.preserve_format).requires_grad_(i == which) for i, t in enumerate(inputs)]
            with torch.no_grad():
                assert not call(*leaves).requires_grad
            out = call(*leaves)
            assert out.requires_grad and torch.equal(out, want)
            with pytest.raises(RuntimeError, match="no autograd formula"):
                out.float().sum().backward()
            with forward_ad.dual_level():
                leaves[which] = forward_ad.make_dual(inputs[which], torch.ones_like(inputs[which]))
                for mode in (torch.no_grad, torch.enable_grad):
                    with mode(), pytest.raises(RuntimeError, match="tangents"):
                        call(*leaves)
        assert torch.equal(call(*inputs), want) and not want.requires_grad
