"""AdamW over a list of tensors (cleanmarl_amd/adamw.py) against plain evaluations of its rule.

The kernel rounds every product and sum of its rule by itself, so a plain fp32 evaluation in the same order has the same bits: states, scales and
codes are compared exactly against that (plain_step).  Against 64 bits (exact_step) the bars are counted from roundings, U = 2^-24:
m and v: two products, a sum and the rounded factors, 4 U of the terms' sum; p: 12 U of the step and 2 U of p, then half a step of its type.
"""
import ctypes as C
import math
import os
import sys

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

U = 2.0 ** -24
BLOCK = 256
H = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = [1, 3, 4, 255, 256, 257, 1000, 4095, 4096, 4097, 12289, 70001]


def f32(x):
    return float(np.float32(x))


def plain_coef(grads, max_norm, scale=1.0):
    total = sum((g.float() * f32(scale)).double().square().sum() for g in grads)
    norm = float(np.float32(math.sqrt(float(total))))
    return norm, min(1.0, f32(np.float32(max_norm) / (np.float32(norm) + np.float32(1e-6))))


def plain_step(p, g, m, v, step, coef=1.0, grad_scale=1.0, h=H):
    """One tensor, 32-bit arithmetic in the kernel's order: (p in fp32, m, v)."""
    b1, b2 = h["betas"]
    g = (g.float() * f32(grad_scale)) * coef
    m = m * f32(b1) + g * f32(1 - b1)
    v = v * f32(b2) + (g * f32(1 - b2)) * g
    denom = torch.sqrt(v) * f32(1 / math.sqrt(1 - b2 ** step)) + f32(h["eps"])
    return p.float() * f32(1 - h["lr"] * h["weight_decay"]) - (m / denom) * f32(h["lr"] / (1 - b1 ** step)), m, v


def encode(m, root):
    """Blocks of 256: (codes of m, codes of the root, scales [blocks][2])."""
    n = m.numel()
    pad = lambda t: torch.nn.functional.pad(t, (0, -n % BLOCK)).view(-1, BLOCK)  # noqa: E731
    m, root = pad(m), pad(root)
    top = torch.stack([m.abs().amax(1), root.amax(1)], 1)
    scale = torch.where(top < 2.0 ** -100, 0.0, top * f32(1 / 448))
    back = torch.where(scale > 0, 1.0 / scale, 0.0)
    code = root * back[:, 1:]
    code = torch.where((code > 0) & (code < 2.0 ** -9), 2.0 ** -9, code)
    return (m * back[:, :1]).to(torch.float8_e4m3fn).view(-1), code.to(torch.float8_e4m3fn).view(-1), scale


def decode(code, scale, column, n):
    return (code.float().view(-1, BLOCK) * scale[:, column:column + 1]).view(-1)[:n]


def exact_step(p, g, m, v, step, coef, h=H):
    b1, b2 = h["betas"]
    p, g, m, v = p.double(), g.double() * coef, m.double(), v.double()
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    u = h["lr"] / (1 - b1 ** step) * m2 / ((v2 / (1 - b2 ** step)).sqrt() + h["eps"])
    return p * (1 - h["lr"] * h["weight_decay"]) - u, m2, v2, b1 * m.abs() + (1 - b1) * g.abs(), u


def tensors(sizes, dtypes, seed, scale=1.0, shift=0):
    gen = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        dt = dtypes[i % len(dtypes)]
        out.append((torch.randn(n + shift, generator=gen) * scale).to(dt).cuda()[shift:])
    return out


# ---------------------------------------------------------------------------------------------------------------- refusals (no GPU needed)
def _call(entries=None, **kw):
    from cleanmarl_amd import _native as N
    from cleanmarl_amd.adamw import _ENTRY
    lib = N.load()
    rows = entries if entries is not None else [{}]
    table = np.zeros(max(1, len(rows)), _ENTRY)
    block = 0
    for r, e in zip(table, rows):
        d = dict(param=0x1000, grad=0x2000, copy=0, n=300, block=block, param_dtype=0, grad_dtype=0, copy_dtype=0)
        d.update(e)
        for k, v in d.items():
            r[k] = v
        block = d["block"] + 2
    o = dict(exp_avg=0x10000, exp_avg_sq=0x20000, scale=0x30000, n_blocks=8, lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, max_norm=0.0, grad_scale=1.0,
             out_norm=None, ws=None, ws_bytes=0, step_dev=None, step=1, state_bits=32)
    o.update(kw)
    s = N.AdamW(*[o[k] for k, _ in N.AdamW._fields_])
    rc = lib.cm_adamw_multi_step(table.ctypes.data_as(C.c_void_p), len(rows), C.byref(s), None)
    assert rc == -1
    return lib.cm_last_error().decode()


def test_bad_steps_are_refused():
    assert "state_bits" in _call(state_bits=16)
    assert "step" in _call(step=0)
    assert "NULL" in _call(exp_avg=None) and "NULL" in _call(exp_avg_sq=None) and "NULL" in _call(state_bits=8, scale=None)
    assert "aligned" in _call(exp_avg=0x10004) and "beta" in _call(beta1=1.0) and "beta" in _call(beta2=-0.1) and "eps" in _call(eps=-1.0)
    assert "workspace" in _call(max_norm=1.0) and "workspace" in _call(max_norm=1.0, out_norm=0x100, ws=0x100, ws_bytes=8)
    assert "n=" in _call([dict(n=-1)]) and "dtype" in _call([dict(param_dtype=5)]) and "dtype" in _call([dict(grad_dtype=-1)]) and "dtype" in _call([dict(copy=0x100, copy_dtype=9)])
    assert "NULL" in _call([dict(param=0)]) and "NULL" in _call([dict(grad=0)])
    assert "aligned" in _call([dict(param=0x1002)]) and "aligned" in _call([dict(grad=0x2001, grad_dtype=2)]) and "aligned" in _call([dict(copy=0x2001, copy_dtype=2)])
    assert "begin inside" in _call([{}, dict(block=1)]) and "begin inside" in _call([dict(block=-1)]) and "behind the arena" in _call([dict(block=7)])
    from cleanmarl_amd import _native as N
    lib = N.load()
    assert lib.cm_adamw_multi_step(None, 0, None, None) == -1 and lib.cm_adamw_workspace_bytes(0) == 0
    assert [lib.cm_adamw_state_blocks(n) for n in (-1, 0, 1, 256, 257)] == [0, 0, 1, 1, 2]


def test_wrapper_refuses_what_it_cannot_step():
    from cleanmarl_amd.adamw import MultiAdamW
    with pytest.raises(ValueError, match="CPU"):
        MultiAdamW([torch.zeros(3)])
    with pytest.raises(ValueError, match="empty"):
        MultiAdamW([])


@pytest.mark.gpu
def test_wrapper_refusals_on_the_device():
    from cleanmarl_amd._native import NativeError
    from cleanmarl_amd.adamw import MultiAdamW
    p = torch.zeros(8, 4).cuda()
    for bad in (dict(params=[p, p]), dict(params=[p, p.view(-1)[4:9]]), dict(params=[p.t()]), dict(params=[p.double()]), dict(params=[p], copies=[]), dict(params=[p], copies=[p]),
                dict(params=[p], copies=[torch.zeros(4, 8).cuda()]), dict(params=[p], state_bits=16), dict(params=[p], betas=(1.0, 0.9)), dict(params=[p, torch.zeros(3)])):
        with pytest.raises(ValueError):
            MultiAdamW(**bad)
    o = MultiAdamW([p])
    for bad in ([], [torch.zeros(4, 8).cuda()], [torch.zeros(8, 4)], [torch.zeros(4, 8).cuda().t()], [torch.zeros(8, 4).cuda().double()]):
        with pytest.raises(ValueError):
            o.step(bad)
    q, low = torch.zeros(8, 4).cuda(), torch.zeros(8, 4, dtype=torch.bfloat16).cuda()
    moved = MultiAdamW([q], copies=[low])
    for t in (q, low):  # a tensor that has left the device since
        there, t.data = t.data, t.data.cpu()
        with pytest.raises(ValueError, match="another device"):
            moved.step([torch.zeros(8, 4).cuda()])
        t.data = there
    counted = MultiAdamW([q], capturable=True)
    counted.betas = (1.0, 0.9)
    with pytest.raises(NativeError, match="beta1"):
        counted.step([torch.zeros(8, 4).cuda()])
    assert counted.state_dict()["step"] == counted.steps == 0
    with pytest.raises(AttributeError):
        o.root_avg_sq
    with pytest.raises(ValueError):
        o.load_state(torch.zeros(3).cuda(), torch.zeros(3).cuda())


# ---------------------------------------------------------------------------------------------------------------- one step, many shapes and types
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pd, gd, shift", [([torch.float32], [torch.float32], 0), ([torch.float32, torch.bfloat16], [torch.bfloat16], 0),
                                            ([torch.float16, torch.float32, torch.bfloat16], [torch.float16, torch.float32, torch.float32], 1)])
def test_steps_against_the_rule(bits, pd, gd, shift):
    from cleanmarl_amd.adamw import MultiAdamW
    params = tensors(SIZES, pd, 1, shift=shift)
    copies = [torch.zeros_like(p, dtype=torch.bfloat16) if i % 2 else None for i, p in enumerate(params)]
    opt = MultiAdamW(params, copies=copies, state_bits=bits, max_norm=1.5, **H)
    ms, vs, roots = [], [], []
    for step in range(1, 4):
        grads = tensors(SIZES, gd, 10 + step, scale=0.01, shift=shift)
        norm, coef = plain_coef(grads, 1.5, 2.0)
        assert coef < 1.0
        before = [p.clone() for p in params]
        opt.step(grads, grad_scale=2.0)
        assert abs(opt.norm[0].item() - norm) <= 2 * U * norm and abs(opt.norm[1].item() - coef) <= 2 * U
        coef = opt.norm[1].item()  # its last bit may differ from the host's; from here on everything is exact
        for i, (p0, g) in enumerate(zip(before, grads)):
            n, b = p0.numel(), opt.starts[i]
            at = slice(b * BLOCK, b * BLOCK + n)
            m0 = ms[i][0] if step > 1 else torch.zeros(n).cuda()
            v0 = ms[i][1] if step > 1 else torch.zeros(n).cuda()
            want, m, v = plain_step(p0, g, m0, v0, step, coef, 2.0)
            assert torch.equal(params[i], want.to(p0.dtype)), (step, i)
            if copies[i] is not None:
                assert torch.equal(copies[i], want.to(torch.bfloat16))
            exact, em, ev, terms, u = exact_step(p0, g.float() * 2.0, m0, v0, step, coef)
            bar = 2 * U * exact.abs() + 12 * U * (u.abs() + H["lr"] * 10 * terms / (ev.sqrt() + 1e-12)) + exact.abs() * torch.finfo(p0.dtype).eps / 2 + 1e-30
            bar = bar + 2.0 ** -25 * (p0.dtype == torch.float16)
            assert bool(((params[i].double() - exact).abs() <= bar * 1.01).all()), (step, i)
            if bits == 32:
                assert torch.equal(opt.exp_avg[at], m) and torch.equal(opt.exp_avg_sq[at], v)
                assert bool(((m.double() - em).abs() <= 4 * U * terms + 1e-40).all()) and bool(((v.double() - ev).abs() <= 5 * U * ev + 1e-40).all())
                state = (m, v)
            else:
                cm, cr, scale = encode(m, torch.sqrt(v))
                blocks = slice(b, b + scale.shape[0])
                whole = slice(b * BLOCK, (b + scale.shape[0]) * BLOCK)
                assert torch.equal(opt.scale[blocks], scale)
                assert torch.equal(opt.exp_avg[whole].view(torch.uint8), cm.view(torch.uint8)) and torch.equal(opt.root_avg_sq[whole].view(torch.uint8), cr.view(torch.uint8))
                dm, dr = decode(cm, scale, 0, n), decode(cr, scale, 1, n)
                # e4m3: half a step is 2^-4 of the value, half of the smallest code's distance 2^-10 of the scale; the smallest root code is rounded up to
                each = scale.repeat_interleave(BLOCK, 0)[:n]
                assert bool(((dm - m).abs() <= m.abs() * 2.0 ** -4 + each[:, 0] * 2.0 ** -10 + 1e-30).all())
                assert bool(((dr - v.sqrt()).abs() <= v.sqrt() * 2.0 ** -4 + each[:, 1] * 2.0 ** -9).all())
                assert bool((dr[(v.sqrt() > 0) & (each[:, 1] > 0)] > 0).all())
                state = (dm, dr * dr)
            ms[i:i + 1] = [state]
        used = torch.zeros(opt.starts[-1] * BLOCK, dtype=torch.bool)
        for i, n in enumerate(SIZES):
            used[opt.starts[i] * BLOCK:opt.starts[i] * BLOCK + n] = True
        assert not opt.exp_avg.float().cpu()[~used].any() and not opt._v.float().cpu()[~used].any()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_long_lists_missing_gradients_and_empty_tensors(bits):
    """More tensors than one launch takes, some without a gradient, some with no elements; those without one keep parameter and states."""
    from cleanmarl_amd.adamw import MultiAdamW
    sizes = [(37 * i) % 600 for i in range(200)]
    params = tensors(sizes, [torch.float32, torch.bfloat16], 5)
    opt = MultiAdamW(params, state_bits=bits, max_norm=0.01, **H)
    state = [(torch.zeros(n).cuda(), torch.zeros(n).cuda()) for n in sizes]
    for step in (1, 2):
        grads = [None if (i + step) % 7 == 0 else g for i, g in enumerate(tensors(sizes, [torch.float32], 20 + step))]
        before = [p.clone() for p in params]
        opt.step(grads)
        norm, _ = plain_coef([g for g in grads if g is not None], 0.01)
        assert abs(opt.norm[0].item() - norm) <= 2 * U * norm
        coef = opt.norm[1].item()
        for i, (p0, g) in enumerate(zip(before, grads)):
            if g is None:
                assert torch.equal(params[i], p0)
                continue
            want, m, v = plain_step(p0, g, *state[i], step, coef)
            assert torch.equal(params[i], want.to(p0.dtype)), (step, i, sizes[i])
            if bits == 8 and m.numel():
                cm, cr, scale = encode(m, v.sqrt())
                m, v = decode(cm, scale, 0, m.numel()), decode(cr, scale, 1, m.numel()).square()
            state[i] = (m, v)
    opt.step([None] * 200)  # nothing to do
    assert opt.norm[0].item() == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_of_more_than_31_bits(bits):
    """Elements behind the 2^31st: the last ones and some in the middle are held to the rule; the norm counts them all."""
    from cleanmarl_amd.adamw import MultiAdamW
    n = (1 << 31) + 777
    p = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    g = torch.full((n,), 2.0 ** -10, dtype=torch.bfloat16, device="cuda")
    spots = [slice(0, 512), slice((1 << 30) - 256, (1 << 30) + 256), slice(n - 777, n)]
    for i, sl in enumerate(spots):
        g[sl] = tensors([sl.stop - sl.start], [torch.bfloat16], i, scale=0.01)[0]
    other = torch.zeros(5, device="cuda")
    opt = MultiAdamW([p, other], state_bits=bits, max_norm=1.0, **H)
    opt.step([g, torch.ones(5, device="cuda")])
    total = float(sum(c.float().double().square().sum() for c in g.split(1 << 28))) + 5
    assert abs(opt.norm[0].item() - math.sqrt(total)) <= 2 * U * math.sqrt(total)
    coef = opt.norm[1].item()
    for sl in spots:
        k = sl.stop - sl.start
        want, m, v = plain_step(torch.full((k,), 0.5, dtype=torch.bfloat16, device="cuda"), g[sl], torch.zeros(k, device="cuda"), torch.zeros(k, device="cuda"), 1, coef)
        assert torch.equal(p[sl], want.to(torch.bfloat16))
    want, _, _ = plain_step(torch.zeros(5, device="cuda"), torch.ones(5, device="cuda"), torch.zeros(5, device="cuda"), torch.zeros(5, device="cuda"), 1, coef)
    assert torch.equal(other, want)


@pytest.mark.gpu
def test_states_of_zero_tiny_and_huge_gradients():
    from cleanmarl_amd.adamw import MultiAdamW
    n = 1024
    for bits in (32, 8):
        p = torch.ones(n).cuda()
        opt = MultiAdamW([p], lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.0, state_bits=bits)
        g = torch.zeros(n).cuda()
        opt.step([g])
        assert bool((p == 1).all()) and not opt._m.float().any()
        g[:256] = 1e-30    # m below every scale, v below fp32: the step is m / eps
        g[256:512] = 1e12
        g[512] = 1.0       # one large value beside small ones: their roots keep a code
        g[513:768] = 1e-7
        for _ in range(3):
            opt.step([g])
        assert bool(torch.isfinite(p).all()) and bool((p[768:] == 1).all()) and bool(((p - 1).abs() <= 3 * 1e-2 * 1.6).all())
        assert bool((p[256:512] < 1).all()) and bool((p[512:768] < 1).all())
        before = p.clone()
        g.zero_()
        opt.step([g])  # the moments alone: no root was rounded away under a moment that was not
        assert bool(((p - before).abs() <= 1e-2 * 1.6).all())
        bad = MultiAdamW([torch.ones(512).cuda()], state_bits=bits, max_norm=1.0)
        g = torch.ones(512).cuda()
        g[300] = math.nan
        bad.step([g])
        assert bool(bad.params[0].isnan().all()) and math.isnan(bad.norm[0].item())  # a norm that is not a number is not hidden
        for value in (math.nan, math.inf):
            one = MultiAdamW([torch.ones(512).cuda()], state_bits=bits)
            g = torch.ones(512).cuda()
            g[300] = value
            one.step([g])
            assert one.params[0].isnan().nonzero().view(-1).tolist() == [300]
            one.step([torch.ones(512).cuda()])
            assert bool(one.params[0][300].isnan()) and bool(torch.isfinite(one.params[0][:256]).all())


@pytest.mark.gpu
def test_agrees_with_the_flat_step():
    """The same numbers as cm_optimizer_step's AdamW on one flat vector.  That one rounds 1 - beta to fp32 from the fp32 beta (2^-25 of it: 2^-25 / 0.01
    relative in the factor of v, half of that in its root) and divides by sqrt(1 - beta2^t) and 1 - beta1^t: 2^-18 of the step holds them."""
    from cleanmarl_amd import _native as N
    from cleanmarl_amd.adamw import MultiAdamW
    lib, n = N.load(), 5000
    p, g = tensors([n], [torch.float32], 3)[0], tensors([n], [torch.float32], 4)[0]
    mine = p.clone()
    opt = MultiAdamW([mine], **H)
    m, v, norm = (torch.zeros(k).cuda() for k in (n, n, 1))
    scr = torch.zeros(lib.cm_opt_step_scratch_bytes(), dtype=torch.uint8).cuda()
    buf = torch.cat([g, torch.zeros(8).cuda()])
    for step in (1, 2, 3):
        buf[:n], buf[n + N.STAT_COUNT] = g, 1.0
        o = N.OptStep(p.data_ptr(), m.data_ptr(), v.data_ptr(), norm.data_ptr(), scr.data_ptr(), H["lr"], 0.9, 0.99, 1e-8, 0.1, 0.0, 1.0, step, N.OPT_ADAMW, None)
        N.check(lib.cm_optimizer_step(buf.data_ptr(), n, C.byref(o), N.stream_ptr()), "cm_optimizer_step")
        opt.step([g])
        assert bool(((p - mine).abs() <= H["lr"] * 2.0 ** -18 * step + 4 * U * p.abs() * step).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoint_and_graph(bits):
    from cleanmarl_amd.adamw import MultiAdamW
    sizes = [1000, 257, 3]
    start = tensors(sizes, [torch.float32], 1)
    grads = tensors(sizes, [torch.float32], 2)
    make = lambda **kw: MultiAdamW([p.clone() for p in start], state_bits=bits, max_norm=0.5, **H, **kw)  # noqa: E731
    eager, other = make(), make()
    for _ in range(3):
        eager.step(grads)
    saved, at = eager.state_dict(), [p.clone() for p in eager.params]
    for _ in range(2):
        eager.step(grads)
    other.load_state_dict(saved)
    for p, q in zip(other.params, at):
        p.copy_(q)
    for _ in range(2):
        other.step(grads)
    assert saved["step"] == 3 and all(torch.equal(a, b) for a, b in zip(eager.params, other.params))
    # a captured step counts on at each replay; two graphs of two optimisers, eager work between the replays
    opts, graphs = [make(capturable=True), make(capturable=True)], []
    for o in opts:
        o.step(grads)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o.step(grads)
        graphs.append(g)
    check = make()
    check.step(grads)
    for k in range(4):
        check.step(grads)
        for g, o in zip(graphs, opts):
            g.replay()
            torch.cuda.synchronize()
        for o in opts:
            for a, b in zip(o.params, check.params):
                assert bool(((a - b).abs() <= 4 * U * (k + 2) * (1 + b.abs())).all()), k
            assert o.step_dev.item() == k + 2


# ---------------------------------------------------------------------------------------------------------------- the operators together
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_training_run_of_a_token_policy(bits):
    """Score with the policy, clipped policy loss, backward through the caller's model, step -- and the same for a preference loss.  The gradients are
    held to autograd's in 64 bits through the same model."""
    from cleanmarl_amd import token_loss as TL
    from cleanmarl_amd.adamw import MultiAdamW
    gen = torch.Generator().manual_seed(0)
    V, D, rows = 1003, 32, 48
    h = torch.randn(rows, D, generator=gen)
    W, b = (torch.randn(V, D, generator=gen) * 0.2), torch.zeros(V)
    tok = torch.randint(V, (rows,), generator=gen)
    adv = torch.randn(rows, generator=gen)
    params = [W.clone().cuda().requires_grad_(True), b.clone().cuda().requires_grad_(True)]
    opt = MultiAdamW([p.data for p in params], lr=1e-2, state_bits=bits, max_norm=1.0)
    hd, tokd, advd = h.cuda(), tok.cuda(), adv.cuda()
    weight = torch.full((rows,), 1.0 / rows).cuda()
    seq = torch.tensor([0, 10, 24, 30, 48], dtype=torch.int32).cuda()
    with torch.no_grad():
        old = TL.token_logprob(hd @ params[0].t() + params[1], tokd).logp
    ref_sum = torch.stack([old[a:e].sum() for a, e in ((0, 10), (10, 24), (24, 30), (30, 48))])
    for it in range(4):
        for p in params:
            p.grad = None
        logits = hd @ params[0].t() + params[1]
        if it % 2 == 0:
            r = TL.policy_loss_fwd_bwd(logits.detach(), tokd, old, advd, logp_ref=old, weight=weight, kl_coef=0.05, entropy_coef=0.01)
        else:
            r = TL.preference_loss_fwd_bwd(logits.detach(), tokd, seq, ref_sum)
        logits.backward(r.dlogits)
        # the same loss in 64 bits
        P = [p.detach().double().requires_grad_(True) for p in params]
        lp_all = torch.log_softmax(hd.double() @ P[0].t() + P[1], 1)
        lp = lp_all[torch.arange(rows), tokd]
        if it % 2 == 0:
            rho = (lp - old.double()).exp()
            d = old.double() - lp
            row = -torch.minimum(advd.double() * rho, advd.double() * rho.clamp(0.8, 1.2)) + 0.05 * (d.exp() - 1 - d) - 0.01 * -(lp_all.exp() * lp_all).sum(1)
            loss = (row * weight.double()).sum()
        else:
            L = torch.stack([lp[a:e].sum() for a, e in ((0, 10), (10, 24), (24, 30), (30, 48))]) - ref_sum.double()
            loss = -torch.nn.functional.logsigmoid(0.1 * (L[:2] - L[2:])).mean()
        want = torch.autograd.grad(loss, P)
        got_loss = float(r.stats[0]) / 2 if it % 2 else float(r.stats[4])
        assert abs(got_loss - float(loss.detach())) <= 1e-5 * (1 + abs(float(loss.detach())))
        for p, w in zip(params, want):  # fp32 products of 48 rows and 32 columns on both sides of kernels good to some 1e-6
            assert float((p.grad.double() - w).norm() / w.norm()) <= 2e-5
        before = [p.detach().clone() for p in params]
        opt.step([p.grad for p in params])
        assert all(bool(torch.isfinite(p).all()) and not torch.equal(p.detach(), q) for p, q in zip(params, before))


# ---------------------------------------------------------------------------------------------------------------- values that leave fp32
@pytest.mark.gpu
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan, 1e22, -3e38])
def test_an_overflow_stays_with_its_element(value):
    """8-bit states: the elements beside one whose moments are not finite (with 1e22 only the second: 1e22^2 / 1000 is beyond fp32) do what they do beside a
    zero gradient, bit for bit, and the element itself does what it does with 32-bit states.  512 elements share the first two blocks; 300 is in the second."""
    from cleanmarl_amd.adamw import MultiAdamW
    n, at = 700, 300
    start = tensors([n], [torch.float32], 1)[0]
    grads = [tensors([n], [torch.float32], 10 + k)[0] for k in range(4)]
    runs = {}
    for name, bits, there in (("8", 8, value), ("beside a zero", 8, 0.0), ("32", 32, value)):
        opt = MultiAdamW([start.clone()], state_bits=bits, lr=1e-2, betas=(0.9, 0.999), weight_decay=0.1)
        steps = []
        for k, g in enumerate(grads):
            g = g.clone()
            g[at] = there if k == 1 else 0.0  # an ordinary step, the value, two more steps
            opt.step([g])
            steps.append(opt.params[0].clone())
        runs[name] = steps
        if name == "8":
            assert bool(torch.isfinite(opt.scale).all())
    others = torch.arange(n, device="cuda") != at
    for got, beside, wide in zip(runs["8"], runs["beside a zero"], runs["32"]):
        assert bool(torch.isfinite(got[others]).all())
        assert torch.equal(got[others], beside[others])
        assert torch.equal(got[at], wide[at]) or (bool(got[at].isnan()) and bool(wide[at].isnan())), (got[at].item(), wide[at].item())
    assert bool(torch.isfinite(runs["8"][-1][at])) == (abs(value) == 1e22 or abs(value) == 3e38)


# ---------------------------------------------------------------------------------------------------------------- autograd
@pytest.mark.gpu
def test_a_step_is_seen_by_graphs_that_saved_a_parameter():
    """As with torch's own in-place operations: a backward pass that needs a parameter or a copy as it was before the step says so."""
    from cleanmarl_amd.adamw import MultiAdamW
    p = torch.ones(8, 4, device="cuda").requires_grad_(True)
    low = torch.ones(8, 4, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    other = torch.ones(3, device="cuda")
    opt = MultiAdamW([p, other], copies=[low, None])
    x = torch.ones(4, 8, device="cuda", requires_grad=True)
    for saved in (x @ p, x.to(torch.bfloat16) @ low):
        opt.step([torch.ones_like(p.detach()), None])
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            saved.sum().backward()
    versions = [t._version for t in (p, low, other)]
    opt.step([None, torch.ones(3, device="cuda")])
    assert [t._version - v for t, v in zip((p, low, other), versions)] == [0, 0, 1]  # what was not written is as it was
    (x @ p).sum().backward()
    assert bool(torch.isfinite(x.grad).all())
    with torch.inference_mode():
        frozen = torch.ones(4, device="cuda")
    o = MultiAdamW([frozen, torch.ones(4, device="cuda")])  # tensors made in inference mode count no versions
    o.step([torch.ones(4, device="cuda")] * 2)
    assert o.steps == 1 and bool((frozen < 1).all())


def test_a_step_without_any_gradient_is_an_error():
    """The default gradients are the parameters' own; where none has one (tensors detached from the parameters never do) nothing would be trained."""
    from cleanmarl_amd.adamw import MultiAdamW
    opt = MultiAdamW.__new__(MultiAdamW)  # (the constructor needs a GPU, the refusal does not)
    opt.params, opt.device, opt.steps = [torch.zeros(3), torch.zeros(4)], torch.device("cuda:0"), 5
    with pytest.raises(ValueError, match="no parameter has a gradient"):
        opt.step()
    assert opt.steps == 5


@pytest.mark.gpu
def test_steps_from_the_parameters_own_gradients():
    from cleanmarl_amd.adamw import MultiAdamW
    p, q = (torch.ones(5, device="cuda").requires_grad_(True) for _ in range(2))
    opt = MultiAdamW([p, q], capturable=True)
    with pytest.raises(ValueError, match="no parameter has a gradient"):
        opt.step()
    assert opt.steps == 0 and opt.step_dev.item() == 0
    p.sum().backward()
    opt.step()  # one of them has one
    assert opt.steps == 1 and bool((p < 1).all()) and bool((q == 1).all())
    opt.step([None, None])  # said so by the caller
    assert opt.steps == 2


def test_a_tensor_of_more_workgroups_than_a_launch_has_is_refused():
    """A launch ends at 2^32 threads, 2^24 workgroups of 256, each of 4096 elements: 2^36 elements are one too many workgroup."""
    last = (1 << 36) - 4096  # 2^24 - 1 workgroups
    for n in (1 << 36, last + 1):
        assert "elements of one tensor" in _call([dict(n=n)], n_blocks=1 << 30)
    assert "aligned" in _call([dict(n=last, grad=0x2001)], n_blocks=1 << 30)  # refused for something else
