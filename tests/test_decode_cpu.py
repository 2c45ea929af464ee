"""CPU checks of the few-token layer and router: refusals (no GPU is touched), shape functions, the sum over expert-parallel ranks."""
import os

import pytest
import torch

P = 1 << 20   # an aligned address that is never dereferenced


def test_layer_entry_point_refuses():
    from mok import _native as nat
    L = nat.lib()

    def call(x=P, xs=256, r=P, w=P, T=4, K=2, H=256, sg=P, su=P, sd=P, si=64, g=P, u=P, d=P, gs=None, us=None, ds=None, I=128, E=8, first=0,
             out=P, scratch=P):
        return L.mok_moe_decode(x, xs, r, w, T, K, H, sg, su, sd, si, g, u, d, gs, us, ds, I, E, first, 0, 0.0, out, scratch, None, None)
    for bad in (dict(x=None), dict(r=None), dict(w=None), dict(g=None), dict(u=None), dict(d=None), dict(out=None), dict(scratch=None), dict(T=0),
                dict(K=0), dict(H=96), dict(H=0), dict(I=32), dict(I=0), dict(si=32), dict(si=-64), dict(E=0), dict(first=-1), dict(su=None),
                dict(sd=None), dict(sg=None), dict(si=0), dict(sg=None, su=None, sd=None), dict(gs=P), dict(gs=P, us=P), dict(us=P), dict(x=P + 8),
                dict(g=P + 2), dict(xs=250), dict(sg=P + 8), dict(scratch=P + 8)):
        assert call(**bad) == -1, bad
    for large in (dict(T=257), dict(K=33), dict(T=256, K=17), dict(E=1025)):
        assert call(**large) == -4, large
    assert L.mok_moe_decode_scratch_bytes(4, 2, 256, 128, 64, 0) == 2 * (4 * 2 * 128 + 4 * 64)
    assert L.mok_moe_decode_scratch_bytes(4, 2, 256, 128, 64, 1) == 2 * (4 * 2 * 128 + 4 * 64) + 2 * 4 * 256 + 4 * (4 + 8)
    assert L.mok_moe_decode_scratch_bytes(0, 2, 256, 128, 64, 0) == 0


def test_router_entry_point_refuses():
    from mok import _native as nat
    L = nat.lib()

    def call(x=P, xs=256, w=P, T=4, H=256, E=8, K=2, logits=P, r=P, rw=P):
        return L.mok_router_decode(x, xs, w, 1, None, T, H, E, K, logits, r, rw, None)
    for bad in (dict(x=None), dict(w=None), dict(logits=None), dict(r=None), dict(rw=None), dict(T=0), dict(H=4), dict(E=0), dict(K=0), dict(K=9),
                dict(E=64, K=33), dict(x=P + 4), dict(w=P + 8), dict(xs=12)):
        assert call(**bad) == -1, bad
    assert call(T=257) == -4 and call(E=1025) == -4


def test_python_calls_refuse():
    import mok
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    r, w = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    g, d = torch.zeros(3, 128, 256, dtype=torch.bfloat16), torch.zeros(3, 256, 128, dtype=torch.bfloat16)
    none = (None,) * 3
    with pytest.raises(ValueError, match="CUDA"):
        mok.moe_decode(x, r, w, *none, g, g, d)
    with pytest.raises(ValueError, match="at most 256"):
        mok.moe_decode(torch.zeros(257, 256, dtype=torch.bfloat16), r, w, *none, g, g, d)
    with pytest.raises(ValueError, match="multiple of 64"):
        mok.moe_decode(x[:, :100], r, w, *none, g, g, d)
    with pytest.raises(ValueError, match="CUDA"):
        mok.route_decode(x, torch.zeros(8, 256), topk=2)


def test_shape_functions():
    import mok  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(5, 256, dtype=torch.bfloat16)
        r, w = torch.ops.mok.router_decode(x, torch.empty(8, 256), None, 3)
        assert (r.shape, r.dtype, w.shape, w.dtype) == ((5, 3), torch.int32, (5, 3), torch.float32)
        g, d = torch.empty(8, 128, 256, dtype=torch.bfloat16), torch.empty(8, 256, 128, dtype=torch.bfloat16)
        out = torch.ops.mok.moe_decode(x, r, w, None, None, None, g, None, g, None, d, None, 0, None)
        assert (out.shape, out.dtype) == ((5, 256), torch.bfloat16)


def _rank(rank, world, port, results):
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    sys.path.insert(0, os.path.join(root, "mixture-of-kittens_b200"))
    import torch.distributed as dist
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world)
    import mok
    from mok import module

    def route(x, w, bias=None, *, topk):
        v, i = torch.topk(x.float() @ w.t(), topk, dim=1)
        return i.to(torch.int32), torch.softmax(v, dim=1)

    def decode(x, routes, weights, sg, su, sd, g, u, d, *, first_expert, swiglu_limit):   # the kernel's formula on the CPU
        out = torch.zeros(x.shape)
        if sg is not None:
            out += (torch.nn.functional.silu(x.float() @ sg.float().t()) * (x.float() @ su.float().t())) @ sd.float().t()
        for e in range(g.shape[0]):
            h = torch.nn.functional.silu(x.float() @ g[e].float().t()) * (x.float() @ u[e].float().t())
            out += (h @ d[e].float().t()) * ((routes == first_expert + e) * weights).sum(1, keepdim=True)
        return out.to(x.dtype)
    module.route_decode, module.moe_decode = route, decode
    torch.manual_seed(0)
    whole = mok.MoKMoE(64, 64, 4, 2, group=dist.new_group([rank], use_local_synchronization=True)) if rank == 0 else None
    torch.manual_seed(0)
    layer = mok.MoKMoE(64, 64, 4, 2)
    torch.manual_seed(0)
    full = [torch.randn(4, 64, 64).mul_(0.2).to(torch.bfloat16) for _ in range(3)]
    x = torch.randn(6, 64).to(torch.bfloat16)
    with torch.no_grad():
        for m, part in ((layer, slice(2 * rank, 2 * rank + 2)), (whole, slice(0, 4))):
            if m is not None:
                for p, w in zip((m.w_routed_gate, m.w_routed_up, m.w_routed_down), full):
                    p.copy_(w[part])
    with torch.no_grad():
        for p in (layer.router, layer.w_shared_gate, layer.w_shared_up, layer.w_shared_down):
            dist.broadcast(p, 0)
        if whole is not None:
            for a in ("router", "w_shared_gate", "w_shared_up", "w_shared_down"):
                getattr(whole, a).copy_(getattr(layer, a))
    out = layer.decode(x)
    results.put((rank, out.float().tolist(), whole.decode(x).float().tolist() if whole is not None else None))
    dist.barrier()
    dist.destroy_process_group()


def test_module_sums_over_ranks():
    import torch.multiprocessing as mp
    ctx = mp.get_context("spawn")
    results = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, 2, 29611 + os.getpid() % 300, results)) for r in range(2)]
    for p in procs:
        p.start()
    got = {r: (o, w) for r, o, w in (results.get(timeout=120) for _ in procs)}
    for p in procs:
        p.join(60)
        assert p.exitcode == 0
    a, b, want = torch.tensor(got[0][0]), torch.tensor(got[1][0]), torch.tensor(got[0][1])
    assert torch.equal(a, b)
    # two parts of half the terms, each rounded to bf16 (2^-8), their sum rounded once more
    assert bool(((a - want).abs() <= 2.0 ** -8 * 3 * (want.abs().max() + 1)).all()) and (a - want).norm() <= 0.02 * want.norm()


def test_tangents_are_refused():
    import mok
    from torch.autograd import forward_ad
    x, w = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(8, 256)
    r, weights = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    g, d = torch.zeros(3, 128, 256, dtype=torch.bfloat16), torch.zeros(3, 256, 128, dtype=torch.bfloat16)
    s = torch.zeros(4, 2)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: mok.route_decode(dual(x), w, topk=2), lambda: mok.route_decode(x, w, dual(w[:, 0].contiguous()), topk=2),
                     lambda: mok.moe_decode(x, r, dual(weights), None, None, None, g, g, d),
                     lambda: mok.moe_decode(x, r, weights, None, None, None, g, g, dual(d)),
                     lambda: mok.rms_norm_quantized(x, dual(w[0])), lambda: mok.block_matmul((x, dual(s)), (x, s))):
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangents"):
                call()
