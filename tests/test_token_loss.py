"""Token-level losses (cleanmarl_amd/token_loss.py) against plain 64-bit evaluations of the same formulas.

Tolerances are counted from roundings (U = 2^-24, half a step of fp32 at 1):
  * t = (x - m) / T carries <= 3 U relative (difference, reciprocal temperature, product); with v_exp_f32 good to 2 U and sum p |t| <= log V, a
    thread's sum of n terms and the <= 24 merges behind it put  U (3 log V + 4 + n + 24)  on s;
  * log p_token = t - log s: that, plus 3 U |t| + 2 U log s + U |log p|;  H = log s - u / s: u's terms carry the same again times their |t|;
  * p_j = e^t / s of a gradient does without the low part of log2(e) / T (up to 2 U of it): 2 U more on |t|, and 2 U * 16 where the reference
    point of the sums lags its largest 16 (in powers of two) behind the row's maximum;
  * a gradient entry: the relative errors of its factors, then one rounding to the logits' type, finfo.eps / 2 of the value.
n is counted as V / 64 + 16: no kernel gives one thread more than that.
"""
import ctypes as C
import math
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
LOWEST = {t: torch.finfo(t).min for t in DTYPES}
SHAPES = [(1, 1), (5, 2), (130, 5), (67, 9), (33, 16), (19, 17), (40, 64), (9, 65), (21, 100), (6, 255), (7, 1000), (5, 2049), (3, 8200), (2, 33001), (3, 65536),
          (2, 131072), (1, 140003), (300, 4100)]


# ---------------------------------------------------------------------------------------------------------------- 64-bit reference
def reference(x, token, avail, T):
    """Per row: (t, p, log p, H, live) in float64 on the CPU; x the logits as they are."""
    z = x.double().cpu()
    if avail is not None:
        z = torch.where(avail.cpu() != 0, z, -math.inf)
    m = z.amax(1, keepdim=True)
    live = (token.cpu() >= 0) & (m[:, 0] != -math.inf)
    t = (z - torch.where(m == -math.inf, 0.0, m)) / T
    e = torch.exp(t)
    logs = torch.log(e.sum(1, keepdim=True))
    lp = t - logs
    p = torch.exp(lp)
    H = -(torch.where(p > 0, p * lp, 0.0)).sum(1)
    return t, p, lp, torch.where(live, H, 0.0), logs, live


class Bars:
    """The tolerances of one problem."""

    def __init__(self, ref, V, token):
        t, p, lp, H, logs, live = ref
        self.s = U * (3 * math.log(max(V, 2)) + 4 + V / 64 + 16 + 24)
        at = token.cpu().clamp(min=0).long()[:, None]
        tt = t.gather(1, at)[:, 0]
        tt = torch.where(tt == -math.inf, 0.0, tt)
        self.logp = torch.where(live, self.s + 3 * U * tt.abs() + 2 * U * logs[:, 0] + U * lp.gather(1, at)[:, 0].abs(), 0.0)
        self.H = torch.where(live, 2 * self.s * (1 + logs[:, 0]) + 4 * U * (H + logs[:, 0]) + 4 * U, 0.0)
        self.p = self.s + 5 * U * torch.where(p > 0, t.abs(), 0.0) + (4 + 32) * U  # relative error of p_j


def rounded(want, dtype):
    """One rounding to dtype: half a step of the value, half of the smallest subnormal."""
    f = torch.finfo(dtype)
    return want.abs() * f.eps / 2 * (1 + 1e-3) + f.smallest_normal * f.eps / 2


def grad_reference(ref, token, g, h, T):
    t, p, lp, H, logs, live = ref
    at = token.cpu().clamp(min=0).long()[:, None]
    one = torch.zeros_like(p).scatter_(1, at, 1.0)
    one = torch.where(t == -math.inf, 0.0, one)
    lpz = torch.where(p > 0, lp, 0.0)
    d = (g[:, None] * (one - p) + h[:, None] * p * (lpz + H[:, None])) / T
    return torch.where(live[:, None], d, 0.0)


def grad_bar(ref, bars, token, g, h, g_rel, T, want, dtype):
    """g_rel: relative error of g per row (what the row's scalars carry)."""
    t, p, lp, H, logs, live = ref
    at = token.cpu().clamp(min=0).long()[:, None]
    one = torch.zeros_like(p).scatter_(1, at, 1.0)
    lpz = torch.where(p > 0, lp, 0.0)
    a = g.abs()[:, None] * (one + p) * (bars.p + g_rel[:, None] + 6 * U)
    b = h.abs()[:, None] * p * ((lpz.abs() + H[:, None]) * (bars.p + 8 * U) + bars.H[:, None] + bars.s + 3 * U * (lpz.abs() + logs))
    flushed = 2.0 ** -126 * (1 + g.abs()[:, None] + h.abs()[:, None] * (lpz.abs() + H[:, None]))  # v_exp_f32 gives 0 for what is below 2^-126
    bar = (a + b + flushed) / T
    return bar + rounded(want.abs() + bar, dtype)


def close(got, want, bar, what):
    got, want = got.double().cpu(), want.double().cpu()
    same = (got == want) | ((got - want).abs() <= bar) | (got.isnan() & want.isnan())
    assert bool(same.all()), f"{what}: {int((~same).sum())} of {same.numel()} off, worst {float(((got - want).abs() / (bar + 1e-300)).nan_to_num(1e30).max()):.3g} bars"


def problem(rows, V, dtype, seed, avail=False, token_dtype=torch.int64, pad=0, shift=0, ignore=True):
    """Logits with a row stride V + pad, starting `shift` elements into an allocation; some tokens negative, some rows without a column."""
    gen = torch.Generator().manual_seed(seed)
    store = torch.full((rows * (V + pad) + shift + 8,), math.nan, dtype=dtype)
    x = store[shift:shift + rows * (V + pad)].view(rows, V + pad)[:, :V] if rows else store[:0].view(0, V)
    x.copy_((torch.randn(rows, V, generator=gen) * 3).to(dtype))
    token = torch.randint(V, (rows,), generator=gen)
    mask = None
    if avail:
        mask = (torch.rand(rows, V, generator=gen) < 0.6).to(torch.uint8)
        mask.scatter_(1, token[:, None], 1)
        odd = torch.tensor([math.nan, math.inf, -math.inf, LOWEST[dtype]], dtype=dtype)[torch.randint(4, (rows, V), generator=gen)]
        x.copy_(torch.where(mask != 0, x, odd))
        if rows > 2:
            mask[rows // 2] = 0
    if ignore and rows > 3:
        token[1] = -100
        token[rows - 1] = -1
    store = store.cuda()
    x = store[shift:shift + rows * (V + pad)].view(rows, V + pad)[:, :V]
    return x, token.to(token_dtype).cuda(), None if mask is None else mask.cuda(), gen


# ---------------------------------------------------------------------------------------------------------------- refusals (no GPU needed)
def _rows(**kw):
    from cleanmarl_amd import _native as N
    d = dict(logits=0x10000, ld=8, avail=None, avail_ld=0, token=0x8000, rows=4, vocab=8, dtype=N.DTYPE_F32, token_bytes=4, reserved=0, temperature=1.0)
    d.update(kw)
    return N.TokenRows(*[d[k] for k, _ in N.TokenRows._fields_])


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=7), "dtype"), (dict(vocab=0), "vocab"), (dict(rows=-1), "rows"), (dict(logits=None), "NULL"), (dict(token=None), "NULL"), (dict(ld=7), "row stride"),
    (dict(avail=0x100, avail_ld=3), "avail"), (dict(token_bytes=2), "token_bytes"), (dict(logits=0x10002), "aligned"), (dict(token=0x8001), "aligned"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"), (dict(temperature=math.nan), "temperature"), (dict(temperature=math.inf), "temperature"),
    (dict(temperature=1e-31), "temperature")])
def test_bad_rows_are_refused_by_every_call(kw, text):
    from cleanmarl_amd import _native as N
    lib, t, p = N.load(), _rows(**kw), 0x900000
    need = 1 << 30
    for rc in (lib.cm_token_logprob(C.byref(t), p, None, None, p, need, None),
               lib.cm_token_logprob_bwd(C.byref(t), p, None, p, None, p, 8, None),
               lib.cm_token_policy_fwd_bwd(C.byref(t), p, p, None, None, 0.2, 0.2, 0.0, 0.0, p, 8, None, p, p, need, None),
               lib.cm_preference_fwd_bwd(C.byref(t), p, 2, p, 0.1, 0.0, 0, 1.0, p, 8, None, None, p, p, need, None)):
        assert rc == -1 and text in lib.cm_last_error().decode()


def test_bad_calls_are_refused():
    from cleanmarl_amd import _native as N
    lib, t, p, big = N.load(), _rows(), 0x900000, 1 << 30
    x = t.logits
    err = lambda rc: lib.cm_last_error().decode() if rc == -1 else f"rc={rc}"  # noqa: E731
    assert "NULL" in err(lib.cm_token_logprob(None, p, None, None, p, big, None))
    assert "logp" in err(lib.cm_token_logprob(C.byref(t), None, None, None, p, big, None))
    assert "workspace" in err(lib.cm_token_logprob(C.byref(t), p, None, None, p, 8, None))
    assert "keep" in err(lib.cm_token_logprob(C.byref(t), p, None, p + 4, p, big, None))
    bwd = lambda keep=p, H=None, dl=p, dh=None, dx=p, ld=8: err(lib.cm_token_logprob_bwd(C.byref(t), keep, H, dl, dh, dx, ld, None))  # noqa: E731
    assert "keep" in bwd(keep=None) and "d_logp" in bwd(dl=None) and "entropy" in bwd(dh=p) and "NULL dlogits" in bwd(dx=None) and "row stride" in bwd(ld=7)
    assert "overlaps" in bwd(dx=x + 4) and "overlaps" in bwd(dx=x, ld=9) and "overlaps" in bwd(dx=x - 4 * 31) and "aligned" in bwd(dx=p + 2)
    pol = lambda old=p, adv=p, ref=None, lo=0.2, hi=0.2, kl=0.0, dx=p, st=p, ws=p, n=big: err(  # noqa: E731
        lib.cm_token_policy_fwd_bwd(C.byref(t), old, adv, ref, None, lo, hi, kl, 0.0, dx, 8, None, st, ws, n, None))
    assert "logp_old" in pol(old=None) and "adv" in pol(adv=None) and "stats" in pol(st=None) and "clip_low" in pol(lo=1.5) and "clip_low" in pol(lo=-0.1)
    assert "clip_high" in pol(hi=-0.1) and "logp_ref" in pol(kl=0.1) and "workspace" in pol(ws=None) and "workspace" in pol(n=16) and "workspace" in pol(ws=p + 8)
    pref = lambda seq=p, pairs=2, ref=p, beta=0.1, sm=0.0, kind=0, st=p, ws=p, n=big, tt=t: err(  # noqa: E731
        lib.cm_preference_fwd_bwd(C.byref(tt), seq, pairs, ref, beta, sm, kind, 1.0, p, 8, None, None, st, ws, n, None))
    assert "pairs" in pref(pairs=0) and "NULL" in pref(seq=None) and "NULL" in pref(ref=None) and "NULL" in pref(st=None) and "kind" in pref(kind=2)
    assert "beta" in pref(beta=0.0) and "label_smoothing" in pref(sm=0.5) and "label_smoothing" in pref(sm=-0.1) and "label_smoothing" in pref(sm=0.1, kind=1)
    assert "workspace" in pref(ws=None) and "workspace" in pref(n=16)
    assert lib.cm_token_workspace_bytes(-1, 5) == 0 and lib.cm_preference_workspace_bytes(5, 5, 0) == 0


def test_wrapper_refuses_what_it_cannot_run():
    from cleanmarl_amd import token_loss as TL
    x, tok, row = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    with pytest.raises(ValueError, match="CPU"):
        TL.token_logprob(x, tok)
    with pytest.raises(ValueError, match="CPU"):
        TL.policy_loss_fwd_bwd(x, tok, row, row)
    with pytest.raises(ValueError, match="last axis"):
        TL._row_stride(torch.zeros(8, 4).t(), "logits")
    with pytest.raises(ValueError, match="one axis of rows"):
        TL._row_stride(torch.zeros(3, 4, 8).transpose(0, 1), "logits")
    assert TL._row_stride(torch.zeros(3, 4, 8), "x") == 8 and TL._row_stride(torch.zeros(5, 10)[:, :8], "x") == 10 and TL._row_stride(torch.zeros(8), "x") == 8
    assert TL._row_stride(torch.zeros(0, 8), "x") == 8 and TL._row_stride(torch.zeros(6, 8)[::2], "x") == 16 and TL._row_stride(torch.zeros(1, 1, 8).expand(1, 1, 8), "x") == 8
    assert TL._row_stride(torch.zeros(3, 8).expand(2, 3, 8)[0], "x") == 8
    with pytest.raises(ValueError, match="one axis of rows"):
        TL._row_stride(torch.zeros(1, 3, 8).expand(2, 3, 8), "x")


# ---------------------------------------------------------------------------------------------------------------- log-probabilities
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, V", SHAPES)
def test_logprob_forward_and_backward(rows, V, dtype):
    from cleanmarl_amd import token_loss as TL
    for k, (avail, T, entropy, tdt, pad, shift) in enumerate([(False, 1.0, False, torch.int64, 0, 0), (True, 0.7, True, torch.int32, 3, 1)]):
        x, tok, mask, gen = problem(rows, V, dtype, 100 * k + V + rows, avail, tdt, pad, shift)
        ref = reference(x, tok, mask, T)
        bars = Bars(ref, V, tok)
        t, p, lp, H, logs, live = ref
        r = TL.token_logprob(x, tok, avail=mask, temperature=T, entropy=entropy, keep=True)
        want = torch.where(live, lp.gather(1, tok.cpu().clamp(min=0).long()[:, None])[:, 0], 0.0)
        close(r.logp, want, bars.logp + U * want.abs(), "logp")
        assert bool((r.logp.cpu()[~live] == 0).all())
        if entropy:
            close(r.entropy, H, bars.H, "entropy")
        dl, dh = torch.randn(rows, generator=gen), torch.randn(rows, generator=gen)
        h = -dh.double() if entropy else torch.zeros(rows, dtype=torch.float64)
        want = grad_reference(ref, tok, dl.double(), h, T)
        bar = grad_bar(ref, bars, tok, dl.double(), h, torch.zeros(rows, dtype=torch.float64), T, want, dtype)
        got = TL.token_logprob_bwd(x, tok, r, dl.cuda(), d_entropy=dh.cuda() if entropy else None, avail=mask, temperature=T)
        close(got, want, bar, "dlogits")
        if mask is not None:
            assert bool((got.cpu()[mask.cpu() == 0] == 0).all())
        y = x.clone() if pad == 0 else x  # in place: over the logits' own rows, whatever their stride
        out = TL.token_logprob_bwd(y, tok, r, dl.cuda(), d_entropy=dh.cuda() if entropy else None, avail=mask, temperature=T, out=y)
        assert out.data_ptr() == y.data_ptr()
        close(out, want, bar, "dlogits in place")  # (another address may take a row apart differently: the bits are those of an equal alignment)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [3, 40, 700, 5000, 70000])
def test_rows_at_the_edges_of_the_type(V, dtype):
    """Rows of the type's lowest value, of -inf, with one column left, with NaN or +inf in an available place."""
    from cleanmarl_amd import token_loss as TL
    x = torch.zeros(8, V, dtype=dtype)
    x[0] = LOWEST[dtype]
    x[1] = -math.inf
    x[2] = -math.inf
    x[2, V - 1] = 1.5
    x[3, V // 2] = math.nan
    x[4, 0] = math.inf
    x[5] = LOWEST[dtype]
    x[5, V - 1] = -LOWEST[dtype]
    x[6, :] = math.nan
    tok = torch.tensor([0, 0, V - 1, 0, 0, V - 1, 0, V])
    logits = x.cuda()
    r = TL.token_logprob(logits, tok.cuda(), entropy=True, keep=True, temperature=0.5)
    logp, H = r.logp.cpu().tolist(), r.entropy.cpu().tolist()
    bar = U * (3 * math.log(V) + 4 + V / 64 + 40) * 2 * (2 + math.log(V))
    assert abs(logp[0] + math.log(V)) <= bar and abs(H[0] - math.log(V)) <= bar
    assert logp[1] == 0.0 and H[1] == 0.0
    assert abs(logp[2]) <= bar and abs(H[2]) <= bar and abs(logp[5]) <= bar and abs(H[5]) <= bar
    assert all(math.isnan(logp[i]) for i in (3, 4, 6, 7)), logp  # what is not a number is not hidden, and neither is a token behind the vocabulary
    ones = torch.ones(8).cuda()
    d = TL.token_logprob_bwd(logits, tok.cuda(), r, ones, temperature=0.5).float().cpu()
    f = torch.finfo(dtype)
    want = (torch.nn.functional.one_hot(torch.tensor([0]), V)[0].double() - 1.0 / V) * 2
    assert bool(((d[0].double() - want).abs() <= want.abs() * (f.eps / 2 + 2 * bar) + 2 * bar / V + f.smallest_normal * f.eps).all())
    # one column left: s is that column's e^t, so p = e^t (1 / s) is 1 up to the division's and the product's rounding (2 U) and 1 - p, times 1 / T = 2,
    # is at most 4 U from 0 (8 U with a division that is good to 3 U); the other columns are 0
    assert bool((d[1] == 0).all()) and bool((d[2].abs() <= 8 * U).all()) and bool((d[5].abs() <= 8 * U).all())
    assert bool((d[2, :V - 1] == 0).all()) and bool((d[5, :V - 1] == 0).all())
    assert bool(d[3].isnan().all()) and bool(d[6].isnan().all()) and bool(d[7].isnan().any())


@pytest.mark.gpu
def test_logprob_shapes_and_empty_batches():
    from cleanmarl_amd import token_loss as TL
    x = torch.randn(2, 3, 50).cuda()
    tok = torch.randint(50, (2, 3)).cuda()
    r = TL.token_logprob(x, tok, entropy=True)
    flat = TL.token_logprob(x.view(6, 50), tok.view(6), entropy=True)
    assert r.logp.shape == (2, 3) and torch.equal(r.logp.view(6), flat.logp) and torch.equal(r.entropy.view(6), flat.entropy)
    one = TL.token_logprob(x[0, 0], tok[0, 0])
    assert one.logp.shape == () and torch.equal(one.logp, r.logp[0, 0])
    e = TL.token_logprob(x[:0], tok[:0], entropy=True, keep=True)
    assert e.logp.shape == (0, 3) and TL.token_logprob_bwd(x[:0], tok[:0], e, e.logp).shape == (0, 3, 50)
    p = TL.policy_loss_fwd_bwd(x[:0], tok[:0], e.logp, e.logp)
    assert p.stats.tolist() == [0.0] * 8 and p.dlogits.shape == (0, 3, 50)
    z = torch.zeros(2).cuda()
    q = TL.preference_loss_fwd_bwd(x[0, :0], tok[0, :0], torch.zeros(3, dtype=torch.int32).cuda(), z)
    assert abs(q.stats[0].item() - math.log(2)) < 1e-6 and q.margin.tolist() == [0.0]
    for bad in (dict(token=tok.float()), dict(token=tok[0]), dict(logits=x.double()), dict(avail=torch.ones(2, 3, 50).cuda()), dict(avail=torch.ones(3, 50, dtype=torch.uint8).cuda()),
                dict(token=tok.cpu()), dict(logits=x.transpose(1, 2), token=tok)):
        with pytest.raises(ValueError):
            TL.token_logprob(**{**dict(logits=x, token=tok), **bad})
    with pytest.raises(ValueError):
        TL.token_logprob_bwd(x, tok, r, r.logp)  # keep=True was not asked for
    k = TL.token_logprob(x, tok, keep=True)
    with pytest.raises(ValueError):
        TL.token_logprob_bwd(x, tok, k, k.logp, d_entropy=k.logp)
    with pytest.raises(ValueError):
        TL.token_logprob_bwd(x, tok, k, k.logp, out=torch.empty(2, 3, 50, dtype=torch.float16).cuda())


# ---------------------------------------------------------------------------------------------------------------- clipped policy loss
def policy_reference(ref, tok, old, adv, refp, w, lo, hi, kl_coef, ent_coef):
    t, p, lp, H, logs, live = ref
    taken = torch.where(live, lp.gather(1, tok.cpu().clamp(min=0).long()[:, None])[:, 0], 0.0)
    live = live & (w != 0)
    rho = torch.exp(taken - old)
    whole, cut = adv * rho, adv * rho.clamp(1 - lo, 1 + hi)
    pg = torch.minimum(whole, cut)
    g = torch.where(whole <= cut, -whole, 0.0)
    kl = torch.zeros_like(rho)
    if refp is not None:
        d = refp - taken
        kl = torch.expm1(d) - d
        g = g - kl_coef * torch.expm1(d)
    clipped = ((rho < 1 - lo) | (rho > 1 + hi)).double()
    loss = -pg - ent_coef * H + kl_coef * kl
    w = torch.where(live, w, 0.0)
    return dict(live=live, logp=torch.where(live, taken, 0.0), g=w * g, h=w * ent_coef, rho=rho, kl=kl,
                rows=[pg, H, (rho - 1) - (taken - old), clipped, loss, live.double(), kl, torch.ones_like(w)], w=w)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, V", SHAPES)
def test_policy_loss(rows, V, dtype):
    from cleanmarl_amd import token_loss as TL
    for k, (avail, T, kl, ent, pad, shift) in enumerate([(False, 1.0, 0.0, 0.0, 0, 0), (True, 0.7, 0.1, 0.02, 5, 3), (False, 1.3, 0.1, 0.0, 0, 1), (True, 1.0, 0.0, 0.01, 0, 0)]):
        lo, hi = 0.2, 0.3
        x, tok, mask, gen = problem(rows, V, dtype, 31 * k + V + 7 * rows, avail, torch.int64 if k % 2 else torch.int32, pad, shift)
        ref = reference(x, tok, mask, T)
        bars = Bars(ref, V, tok)
        taken = torch.where(ref[5], ref[2].gather(1, tok.cpu().clamp(min=0).long()[:, None])[:, 0], 0.0)
        noise = torch.randn(rows, generator=gen).double() * 0.2
        for border in (math.log(1 - lo), math.log(1 + hi)):  # a ratio next to a border may take either branch
            noise = torch.where((noise - border).abs() < 1e-3, noise + 4e-3, noise)
        old = (taken - noise).float()
        adv = torch.randn(rows, generator=gen)
        refp = (taken + torch.randn(rows, generator=gen) * 0.3).float() if kl else None
        w = torch.rand(rows, generator=gen) + 0.5
        if rows > 6:
            w[4] = 0.0
            adv[5] = 0.0
        want = policy_reference(ref, tok, old.double(), adv.double(), None if refp is None else refp.double(), w.double(), lo, hi, kl, ent)
        cu = lambda v: None if v is None else v.cuda()  # noqa: E731
        r = TL.policy_loss_fwd_bwd(x, tok, cu(old), cu(adv), logp_ref=cu(refp), weight=cu(w), avail=mask, temperature=T, clip_low=lo, clip_high=hi, kl_coef=kl, entropy_coef=ent)
        live = want["live"]
        close(r.logp, want["logp"], bars.logp + U * want["logp"].abs(), "logp")
        delta = bars.logp + U * (want["logp"].abs() + 4)  # absolute error of a log ratio = relative error of a ratio
        whole = (adv.double() * want["rho"]).abs() * want["w"]
        ek = (torch.exp(refp.double() - taken) if kl else torch.zeros(rows, dtype=torch.float64)) * want["w"] * kl
        g_abs = torch.where(live, whole * (delta + 6 * U) + (ek + kl * want["w"]) * (delta + 6 * U), 0.0)
        # absolute error of g as a relative one where g is not zero; where it is (clipped rows) nothing may remain
        g_rel = torch.where(want["g"] != 0, g_abs / want["g"].abs().clamp(min=1e-300), 0.0)
        dwant = torch.where(live[:, None], grad_reference(ref, tok, want["g"], want["h"], T), 0.0)
        bar = grad_bar(ref, bars, tok, want["g"], want["h"], g_rel, T, dwant, dtype)
        close(r.dlogits, dwant, bar, "dlogits")
        # statistics: sums over the live rows of values with these absolute errors, one rounding to fp32
        err_row = dict(zip(range(8), [whole * (delta + 6 * U), want["w"] * bars.H, want["w"] * (want["rho"] * (delta + 4 * U) + delta + 4 * U), 0 * whole,
                                      whole * (delta + 8 * U) + want["w"] * (ent * bars.H + 8 * U) + ek * (delta + 4 * U) + kl * want["w"] * (delta + 4 * U), 0 * whole,
                                      want["w"] * ((want["kl"] + 2) * 2 * (delta + 4 * U)) if kl else 0 * whole, 0 * whole]))

        def check_stats(stats):
            for i in range(8):
                v = want["rows"][i] if i == 5 else want["rows"][i] * want["w"]
                v = torch.where(live, v, 0.0)
                bar_i = float(torch.where(live, err_row[i] + 4 * U * v.abs(), 0.0).sum()) + 2 * U * abs(float(v.sum()))
                assert abs(float(stats[i]) - float(v.sum())) <= bar_i, (i, float(stats[i]), float(v.sum()), bar_i)

        check_stats(r.stats)
        args = dict(logp_ref=cu(refp), weight=cu(w), avail=mask, temperature=T, clip_low=lo, clip_high=hi, kl_coef=kl, entropy_coef=ent)
        again = TL.policy_loss_fwd_bwd(x, tok, cu(old), cu(adv), **args)
        assert torch.equal(again.stats, r.stats) and torch.equal(again.dlogits, r.dlogits)  # the same bits every time
        over = TL.policy_loss_fwd_bwd(x, tok, cu(old), cu(adv), out=x, **args)
        close(over.dlogits, dwant, bar, "dlogits in place")
        check_stats(over.stats)


def _policy_case(x, tok, mask, T, seed, kl=0.1, ent=0.02):
    """Everything of a policy call on given logits but the comparison of its statistics: (result, log-probabilities, gradient, its bar)."""
    from cleanmarl_amd import token_loss as TL
    rows, V = x.shape
    gen = torch.Generator().manual_seed(seed)
    ref = reference(x, tok, mask, T)
    bars = Bars(ref, V, tok)
    live = ref[5]
    taken = torch.where(live, ref[2].gather(1, tok.cpu().clamp(min=0).long()[:, None])[:, 0], 0.0)
    old = (taken - torch.randn(rows, generator=gen).double().clamp(-2, 2) * 0.05).float()
    adv, refp = torch.randn(rows, generator=gen), (taken + 0.3).float()
    want = policy_reference(ref, tok, old.double(), adv.double(), refp.double(), torch.ones(rows).double(), 0.2, 0.2, kl, ent)
    dwant = torch.where(live[:, None], grad_reference(ref, tok, want["g"], want["h"], T), 0.0)
    delta = bars.logp + U * (taken.abs() + 4)
    g_abs = (adv.double() * want["rho"]).abs() * (delta + 6 * U) + (torch.exp(refp.double() - taken) + 1) * kl * (delta + 6 * U)
    g_rel = torch.where(want["g"] != 0, g_abs / want["g"].abs().clamp(min=1e-300), 0.0)
    bar = grad_bar(ref, bars, tok, want["g"], want["h"], g_rel, T, dwant, x.dtype)
    call = lambda out=None: TL.policy_loss_fwd_bwd(x, tok, old.cuda(), adv.cuda(), logp_ref=refp.cuda(), avail=mask, temperature=T, kl_coef=kl, entropy_coef=ent, out=out)  # noqa: E731
    return call, want["logp"], bars.logp + U * want["logp"].abs(), dwant, bar, live


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [3, 40, 700, 5000, 70000, 140002, 170002])
def test_policy_loss_on_rows_of_every_size(V, dtype):
    """Rows beside each other that are ordinary, far from zero, of one value (the type's lowest), with -inf among them, or all -inf; small temperatures."""
    gen = torch.Generator().manual_seed(V)
    x = torch.randn(9, V, generator=gen) * 2
    x[1] = x[1] * 0.5 + (30000 if dtype == torch.float16 else 1e5)
    x[2] = LOWEST[dtype]
    x[3, 1::2] = -math.inf
    x[4] = -math.inf
    x[5] = LOWEST[dtype]
    x[5, 0] = 1.0
    x[6] = x[6] - (30000 if dtype == torch.float16 else 3e4)
    x[7, :] = 0.25
    x = x.to(dtype)
    tok = torch.tensor([0, V - 1, 0, 0, 0, 0, V // 2, V // 2, V - 1])
    tok[6] = int(x[6].float().argmax())
    tok[1] = int(x[1].float().argmax())
    for T in (1.0, 0.01):
        xs, toks = x.cuda(), tok.cuda()
        call, lp, lp_bar, dwant, bar, live = _policy_case(xs, toks, None, T, V, kl=0.0)
        r = call()
        close(r.logp, lp, lp_bar, "logp")
        close(r.dlogits, dwant, bar, "dlogits")
        assert int(r.stats[5]) == int(live.sum()) == 8
        over = call(out=xs)
        close(over.dlogits, dwant, bar, "dlogits in place")


@pytest.mark.gpu
@pytest.mark.parametrize("V, dtype", [(65536, torch.bfloat16), (32768, torch.float32), (65601, torch.float16)])
def test_a_long_batch_in_slices(V, dtype):
    """More rows than workgroups, some left out: the same rows in slices of less than one round give the same values, bit by bit where every row starts at the
    same alignment, else within the bars of both (twice one bar)."""
    from cleanmarl_amd import token_loss as TL
    rows = 2300 if V % 64 == 0 else 1100
    gen = torch.Generator("cuda").manual_seed(V)
    x = torch.randn(rows, V, generator=gen, device="cuda", dtype=dtype)
    tok = torch.randint(V, (rows,), generator=gen, device="cuda")
    tok[torch.rand(rows, generator=gen, device="cuda") < 0.3] = -1
    w = (torch.rand(rows, generator=gen, device="cuda") < 0.8).float()
    mask = (torch.rand(rows, V, generator=gen, device="cuda", dtype=torch.float16) < 0.7).to(torch.uint8) if V % 2 else None
    old, adv = torch.randn(rows, generator=gen, device="cuda") - 12, torch.randn(rows, generator=gen, device="cuda")
    r = TL.policy_loss_fwd_bwd(x, tok, old, adv, weight=w, avail=mask, entropy_coef=0.01)
    total = torch.zeros(8, dtype=torch.float64)
    for a in range(0, rows, 230):
        b = min(rows, a + 230)
        part = TL.policy_loss_fwd_bwd(x[a:b], tok[a:b], old[a:b], adv[a:b], weight=w[a:b], avail=None if mask is None else mask[a:b], entropy_coef=0.01,
                                      out=torch.empty(b - a + 1, V, dtype=dtype, device="cuda")[:b - a] if V % 64 == 0 else None)
        if V % 64 == 0:
            assert torch.equal(part.dlogits, r.dlogits[a:b]) and torch.equal(part.logp, r.logp[a:b])
        else:
            # each side is within U (3 log V + V / 64 + 44 + 5 |t| + 48) of the size of its terms, p (|g| + |h| (|log p| + H)), and rounded once (together one
            # whole step): the entropy's term and the loss's may cancel, so the result's own size is no measure
            s_bar = U * (3 * math.log(V) + V / 64 + 92)
            assert bool(((part.logp == r.logp[a:b]) | ((part.logp - r.logp[a:b]).abs() <= 2 * (s_bar + 40 * U))).all())  # (-inf: a token that is not available)
            z = x[a:b].double().masked_fill(mask[a:b] == 0, -1e5)
            lp = torch.log_softmax(z, 1)
            size = lp.exp() * ((adv[a:b].double() * torch.exp(r.logp[a:b].double() - old[a:b].double())).abs()[:, None] + 0.01 * (lp.abs() + math.log(V)))
            bar = 2 * size * (s_bar + 5 * U * lp.abs().clamp(max=1000)) + torch.finfo(dtype).eps * r.dlogits[a:b].double().abs() * 1.01 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
            assert bool(((part.dlogits.double() - r.dlogits[a:b].double()).abs() <= bar).all())
        total += part.stats.double().cpu()
    dead = (tok < 0) | (w == 0)
    assert bool((r.dlogits[dead] == 0).all()) and bool((r.logp[dead] == 0).all()) and int(r.stats[5]) == rows - int(dead.sum()) - 0
    got = r.stats.double().cpu()  # (an unavailable token makes the divergence infinite on both sides)
    assert bool(((got == total) | ((got - total).abs() <= 1e-5 * (1 + total.abs()))).all())


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows whose distance in elements does not fit 31 bits, and products of row and stride that do not fit 32."""
    from cleanmarl_amd import token_loss as TL
    for V, rows in ((1000, 3), (7, 3)):
        ld = (1 << 31) + 8
        store = torch.empty(ld * (rows - 1) + V, dtype=torch.float16, device="cuda")
        x = store.as_strided((rows, V), (ld, 1))
        small = (torch.randn(rows, V, generator=torch.Generator().manual_seed(V)) * 2).to(torch.float16).cuda()
        x.copy_(small)
        tok, one = torch.tensor([1, 0, V - 1]).cuda(), torch.ones(rows).cuda()
        a, b = TL.token_logprob(x, tok, entropy=True, keep=True), TL.token_logprob(small, tok, entropy=True, keep=True)
        assert bool(((a.logp - b.logp).abs() <= 1e-5).all()) and bool(((a.entropy - b.entropy).abs() <= 1e-5).all())
        want = TL.policy_loss_fwd_bwd(small, tok, b.logp, one)
        da = TL.token_logprob_bwd(x, tok, a, one)
        db = TL.token_logprob_bwd(small, tok, b, one)
        assert bool(((da.float() - db.float()).abs() <= db.float().abs() * 2.0 ** -10 + 2.0 ** -24).all())
        got = TL.policy_loss_fwd_bwd(x, tok, b.logp, one, out=x)
        assert bool(((got.dlogits.float() - want.dlogits.float()).abs() <= want.dlogits.float().abs() * 2.0 ** -10 + 2.0 ** -24).all())
        del store, x, got


@pytest.mark.gpu
def test_policy_gradient_against_differences():
    """Central differences of the loss statistic, one logit at a time.  Step 2^-7: a loss good to 2^-20 gives 2^-13 / 2, the third derivative
    (bounded by ~ 10 here) times step^2 / 6 gives 1e-4: 1e-3 holds both."""
    from cleanmarl_amd import token_loss as TL
    V, step = 7, 2.0 ** -7
    gen = torch.Generator().manual_seed(3)
    x = (torch.randn(1, V, generator=gen) * 8).round() / 8
    tok = torch.tensor([2]).cuda()
    kw = dict(logp_old=torch.tensor([-1.9]).cuda(), adv=torch.tensor([0.7]).cuda(), logp_ref=torch.tensor([-2.1]).cuda(), temperature=0.8, clip_low=0.9, clip_high=9.0, kl_coef=0.3,
              entropy_coef=0.2)
    d = TL.policy_loss_fwd_bwd(x.cuda(), tok, **kw).dlogits.cpu()[0]
    for j in range(V):
        up, down = x.clone(), x.clone()
        up[0, j] += step
        down[0, j] -= step
        diff = (TL.policy_loss_fwd_bwd(up.cuda(), tok, **kw).stats[4] - TL.policy_loss_fwd_bwd(down.cuda(), tok, **kw).stats[4]).item() / (2 * step)
        assert abs(diff - d[j].item()) < 1e-3, (j, diff, d[j].item())


@pytest.mark.gpu
@pytest.mark.parametrize("rows, V", [(5000, 5), (3000, 33), (70000, 2), (2600, 600)])
def test_many_rows(rows, V):
    """More rows than one round of any grid."""
    from cleanmarl_amd import token_loss as TL
    x, tok, mask, gen = problem(rows, V, torch.float32, V, True, torch.int32)
    ref = reference(x, tok, mask, 1.0)
    bars = Bars(ref, V, tok)
    adv = torch.randn(rows, generator=gen)
    taken = torch.where(ref[5], ref[2].gather(1, tok.cpu().clamp(min=0).long()[:, None])[:, 0], 0.0).float()
    r = TL.policy_loss_fwd_bwd(x, tok, taken.cuda(), adv.cuda(), avail=mask)
    close(r.logp, torch.where(ref[5], taken.double(), 0.0), bars.logp + 2 * U * taken.double().abs(), "logp")
    g = torch.where(ref[5], -adv.double() * torch.exp(taken.double() * 0), 0.0)
    want = grad_reference(ref, tok, g, torch.zeros_like(g), 1.0)
    bar = grad_bar(ref, bars, tok, g, torch.zeros_like(g), bars.logp + U * (taken.double().abs() + 8), 1.0, want, torch.float32)
    close(r.dlogits, want, bar, "dlogits")
    assert int(r.stats[5]) == int(ref[5].sum())


# ---------------------------------------------------------------------------------------------------------------- preference loss
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths, V, front, behind", [([1, 1], 5, 0, 0), ([3, 0, 7, 2], 100, 2, 3), ([40, 1, 300, 17, 5, 90], 1030, 0, 5), ([2, 5, 3, 1], 40000, 1, 0), ([(7 * i) % 5 for i in range(1300)], 12, 1, 2), ([1] * 600, 9000, 0, 1), ([600, 500], 64, 0, 9),
                                                        ([2, 1, 1, 3], 140001, 0, 2)])
def test_preference_loss(lengths, V, front, behind, dtype):
    from cleanmarl_amd import token_loss as TL
    P = len(lengths) // 2
    start = torch.tensor([front] + [front + sum(lengths[:i + 1]) for i in range(2 * P)], dtype=torch.int32)
    rows = int(start[-1]) + behind
    for kind, smooth, beta, avail, T, inplace in [("sigmoid", 0.0, 0.1, False, 1.0, False), ("sigmoid", 0.1, 0.3, True, 0.8, False), ("squared", 0.0, 0.2, False, 1.0, True)]:
        x, tok, mask, gen = problem(rows, V, dtype, V + P, avail, torch.int64, pad=1, ignore=True)
        ref = reference(x, tok, mask, T)
        bars = Bars(ref, V, tok)
        live = ref[5]
        logp = torch.where(live, ref[2].gather(1, tok.cpu().clamp(min=0).long()[:, None])[:, 0], 0.0)
        which = torch.full((rows,), -1, dtype=torch.int64)
        for q in range(2 * P):
            which[start[q]:start[q + 1]] = q
        L = torch.stack([logp[which == q].sum() for q in range(2 * P)])
        L_bar = torch.stack([(bars.logp + U * logp.abs())[which == q].sum() for q in range(2 * P)])
        rp = (L + torch.randn(2 * P, generator=gen) * 2).float()
        ratio = L - rp.double()
        margin = ratio[:P] - ratio[P:]
        m_bar = L_bar[:P] + L_bar[P:] + 1e-14 * L.abs().max()
        if kind == "sigmoid":
            z = beta * margin
            loss = -(1 - smooth) * torch.nn.functional.logsigmoid(z) - smooth * torch.nn.functional.logsigmoid(-z)
            d, slope, curve = beta * (smooth * torch.sigmoid(z) - (1 - smooth) * torch.sigmoid(-z)), beta, beta * beta / 4
        else:
            loss, d = (margin - 0.5 / beta) ** 2, 2 * (margin - 0.5 / beta)
            slope, curve = d.abs().max().item(), 2.0
        g = torch.where(which >= 0, torch.cat([d, -d])[which.clamp(min=0)] / P, 0.0)
        g_abs = torch.where(which >= 0, (curve * torch.cat([m_bar, m_bar]))[which.clamp(min=0)] / P + 2 * U * g.abs(), 0.0)
        want = grad_reference(ref, tok, g, torch.zeros_like(g), T)
        g_rel = torch.where(g != 0, g_abs / g.abs().clamp(min=1e-300), 0.0)
        bar = grad_bar(ref, bars, tok, g, torch.zeros_like(g), g_rel, T, want, dtype)
        before = x.clone()
        out = x if inplace else torch.full((rows, V), 7.0, dtype=dtype).cuda()
        untouched = (before if inplace else out.clone())[which.cuda() < 0]
        r = TL.preference_loss_fwd_bwd(x, tok, start.cuda(), rp.cuda(), beta=beta, label_smoothing=smooth, kind=kind, avail=mask, temperature=T, out=out)
        close(r.seq_logp, L, L_bar + U * L.abs(), "seq_logp")
        close(r.margin, margin, m_bar + U * margin.abs(), "margin")
        inside = which >= 0
        close(r.dlogits[inside.cuda()], want[inside], bar[inside], "dlogits")
        assert torch.equal(r.dlogits[which.cuda() < 0].nan_to_num(), untouched.nan_to_num())  # rows in front and behind stay as they were
        wants = [loss.sum(), (margin > 0).double().sum(), margin.sum(), L[:P].sum(), L[P:].sum(), P]
        sbars = [float(m_bar.sum()) * slope, 0.0, float(m_bar.sum()), float(L_bar.sum()), float(L_bar.sum()), 0.0]
        for i, (v, b) in enumerate(zip(wants, sbars)):
            assert abs(float(r.stats[i]) - float(v)) <= b + 2 * U * abs(float(v)) + 1e-12, (i, float(r.stats[i]), float(v), b)
        if not inplace:
            fresh = TL.preference_loss_fwd_bwd(x, tok, start.cuda(), rp.cuda(), beta=beta, label_smoothing=smooth, kind=kind, avail=mask, temperature=T)
            assert torch.equal(fresh.dlogits[inside.cuda()], r.dlogits[inside.cuda()]) and bool((fresh.dlogits[which.cuda() < 0] == 0).all())


@pytest.mark.gpu
def test_preference_loss_far_margins_and_refusals():
    from cleanmarl_amd import token_loss as TL
    x, tok = torch.zeros(2, 4).cuda(), torch.zeros(2, dtype=torch.int64).cuda()
    seq = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    for m in (1e5, -1e5):  # softplus and sigmoid far out: no overflow
        r = TL.preference_loss_fwd_bwd(x, tok, seq, torch.tensor([-m, 0.0]).cuda(), beta=1.0)
        assert abs(r.stats[0].item() - max(-m, 0.0)) <= 1e-3 and bool(torch.isfinite(r.dlogits).all())
    for bad in (dict(seq_start=seq.long()), dict(seq_start=seq[:2]), dict(seq_start=seq.cpu()), dict(logp_ref=torch.zeros(3).cuda()), dict(kind="other"), dict(logits=x[None], token=tok[None])):
        with pytest.raises(ValueError):
            TL.preference_loss_fwd_bwd(**{**dict(logits=x, token=tok, seq_start=seq, logp_ref=torch.zeros(2).cuda()), **bad})


# ---------------------------------------------------------------------------------------------------------------- streams, graphs
@pytest.mark.gpu
def test_calls_on_two_streams_and_in_graphs():
    """Two streams at once, and captured graphs replayed in turn with eager work between: every result is the eager one."""
    from cleanmarl_amd import token_loss as TL
    gen = torch.Generator("cuda").manual_seed(5)
    calls = []
    for rows, V, dtype in ((40, 30001, torch.bfloat16), (300, 700, torch.bfloat16), (5, 131072, torch.float16), (1100, 65536, torch.bfloat16), (900, 6, torch.float32)):
        x = torch.randn(rows, V, generator=gen, device="cuda", dtype=dtype)
        tok = torch.randint(V, (rows,), generator=gen, device="cuda")
        tok[::7] = -1
        old, adv = torch.randn(rows, generator=gen, device="cuda") - 8, torch.randn(rows, generator=gen, device="cuda")
        calls.append(lambda x=x, tok=tok, old=old, adv=adv: TL.policy_loss_fwd_bwd(x, tok, old, adv, clip_high=0.3, entropy_coef=0.01))

        def scored(x=x, tok=tok, adv=adv):
            f = TL.token_logprob(x, tok, entropy=True, keep=True)
            return f.logp, f.entropy, TL.token_logprob_bwd(x, tok, f, adv, d_entropy=adv)
        calls.append(scored)
        seq = torch.tensor([0, rows // 4, rows // 2, rows // 2 + 1, rows], dtype=torch.int32, device="cuda")
        calls.append(lambda x=x, tok=tok, seq=seq: TL.preference_loss_fwd_bwd(x, tok, seq, torch.zeros(4, device="cuda")))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    same = lambda a, b: all(torch.equal(u, v) for u, v in zip(a, b))  # noqa: E731
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(2):
        got = []
        for i, c in enumerate(calls):
            with torch.cuda.stream(streams[i % 2]):
                got.append(c())
        torch.cuda.synchronize()
        assert [same(a, b) for a, b in zip(got, want)] == [True] * len(calls)
    graphs, outs = [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c())
        graphs.append(g)
    for k in range(3):
        for i, g in enumerate(graphs):
            for t in outs[i]:
                t.zero_()
            g.replay()
            calls[(i + 1) % len(calls)]()
            torch.cuda.synchronize()
            assert same(outs[i], want[i]), (k, i)


# ---------------------------------------------------------------------------------------------------------------- autograd
@pytest.mark.gpu
def test_gradients_over_the_logits_are_seen_by_graphs_that_saved_them():
    """``out=`` over the logits: a graph whose last operation saved its output (tanh) can no longer run backward and says so; one that did not (a product) can."""
    from cleanmarl_amd import token_loss as TL
    rows, V = 4, 40
    gen = torch.Generator().manual_seed(1)
    z = torch.randn(rows, V, generator=gen).cuda().requires_grad_(True)
    w = torch.eye(V).cuda()
    tok, row = torch.arange(rows).cuda(), torch.full((rows,), -2.0).cuda()
    seq = torch.tensor([0, 2, 4], dtype=torch.int32).cuda()

    def scored(logits, out):
        f = TL.token_logprob(logits, tok, keep=True)
        return TL.token_logprob_bwd(logits, tok, f, row, out=out)

    for call in (scored, lambda logits, out: TL.policy_loss_fwd_bwd(logits, tok, row, row, out=out).dlogits,
                 lambda logits, out: TL.preference_loss_fwd_bwd(logits, tok, seq, torch.zeros(2).cuda(), out=out).dlogits):
        logits = torch.tanh(z)
        d = call(logits.detach(), logits.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            logits.backward(d)
        logits = torch.tanh(z)
        before = logits._version
        d = call(logits.detach(), None)
        assert logits._version == before
        want, = torch.autograd.grad(logits, z, d)
        assert torch.allclose(want, d * (1 - torch.tanh(z).detach() ** 2), rtol=1e-5, atol=1e-7)
        logits = z @ w
        d = call(logits.detach(), logits.detach())
        got, = torch.autograd.grad(logits, z, d.clone())
        assert torch.equal(got, d)  # (w is the unit matrix)
    with torch.inference_mode():
        frozen = torch.zeros(rows, V, device="cuda")
    assert TL.policy_loss_fwd_bwd(frozen, tok, row, row, out=frozen).dlogits is frozen  # tensors made in inference mode count no versions


# ---------------------------------------------------------------------------------------------------------------- calls that read or write where they must not
def test_outputs_over_inputs_are_refused():
    """The policy loss reads its per-row inputs through the scalar cache and ahead of the rows it writes: an output that lies over one of them (the same place, a part of it,
    or from the other side) is refused; directly in front or behind is not an overlap (then the next refusal is met)."""
    from cleanmarl_amd import _native as N
    lib, big = N.load(), 1 << 30
    t = _rows(avail=0xa0000, avail_ld=8, rows=16)  # 16 rows: 64 bytes of a per-row value, 128 of avail, 512 of logits
    place = dict(old=0x20000, adv=0x21000, ref=0x22000, w=0x23000, logp=0x24000, stats=0x25000, dx=0x30000, ws=0x40000)

    def call(tt=t, clip_low=0.2, **kw):
        a = {**place, **kw}
        rc = lib.cm_token_policy_fwd_bwd(C.byref(tt), a["old"], a["adv"], a["ref"], a["w"], clip_low, 0.2, 0.0, 0.0, a["dx"], 8, a["logp"], a["stats"], a["ws"], big, None)
        assert rc != 0
        return lib.cm_last_error().decode()

    for name in ("old", "adv", "ref", "w"):
        for shift in (0, 60, -60):
            assert "logp overlaps" in call(logp=place[name] + shift), (name, shift)
        for shift in (0, 60, -28):
            assert "stats overlaps" in call(stats=place[name] + shift), (name, shift)
        for shift in (0, 60, -508):
            assert "dlogits overlaps" in call(dx=place[name] + shift), (name, shift)
    assert "logp overlaps" in call(logp=t.token) and "stats overlaps" in call(stats=t.token + 60) and "dlogits overlaps" in call(dx=t.token - 508)
    assert "logp overlaps" in call(logp=t.logits + 508) and "stats overlaps" in call(stats=t.avail + 124) and "dlogits overlaps" in call(dx=t.avail - 508)
    assert "logp overlaps" in call(logp=place["dx"] + 4) and "stats overlaps" in call(stats=place["logp"] + 60) and "stats overlaps" in call(stats=place["dx"] + 508)
    # the other calls
    p, err = 0x900000, lambda rc: lib.cm_last_error().decode() if rc == -1 else f"rc={rc}"  # noqa: E731
    for lp, H, keep, ws, text in ((t.logits, None, None, p, "logp overlaps"), (p, p + 60, None, p + 256, "entropy overlaps"), (p, None, t.avail, p + 256, "keep overlaps"),
                                  (p, None, None, t.token, "the workspace overlaps")):
        assert text in err(lib.cm_token_logprob(C.byref(t), lp, H, keep, ws, big, None))
    bwd = dict(keep=0x20000, H=0x21000, dl=0x22000, dh=0x23000)
    for at in (*bwd.values(), t.token, t.avail):
        assert "dlogits overlaps" in err(lib.cm_token_logprob_bwd(C.byref(t), *bwd.values(), at - 508, 8, None))
    pref = dict(seq=0x20000, ref=0x21000, dx=0x30000, margin=0x24000, sums=0x25000, stats=0x26000, ws=0x400000)

    def pairs(**kw):
        a = {**pref, **kw}
        return err(lib.cm_preference_fwd_bwd(C.byref(t), a["seq"], 2, a["ref"], 0.1, 0.0, 0, 1.0, a["dx"], 8, a["margin"], a["sums"], a["stats"], a["ws"], big, None))

    for name, size in (("seq", 20), ("ref", 16)):
        assert "dlogits overlaps" in pairs(dx=pref[name] - 508) and "margin overlaps" in pairs(margin=pref[name] + size - 4) and "seq_logp overlaps" in pairs(sums=pref[name])
        assert "stats overlaps" in pairs(stats=pref[name] - 28) and "the workspace overlaps" in pairs(ws=pref[name])
    assert "margin overlaps" in pairs(margin=t.logits) and "seq_logp overlaps" in pairs(sums=pref["margin"] + 4) and "stats overlaps" in pairs(stats=t.token)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [40, 9000])
def test_outputs_next_to_inputs_are_not_overlaps(V):
    """Per-row inputs and outputs cut out of one allocation, without a gap, give what separate ones give."""
    from cleanmarl_amd import _native as N
    from cleanmarl_amd import token_loss as TL
    lib, rows = N.load(), 16
    gen = torch.Generator().manual_seed(V)
    x, tok = torch.randn(rows, V, generator=gen).cuda(), torch.randint(V, (rows,), generator=gen).cuda()
    old, adv, ref, w = (torch.rand(rows, generator=gen).cuda() - 5 * (k == 0) for k in range(4))
    want = TL.policy_loss_fwd_bwd(x, tok, old, adv, logp_ref=ref, weight=w, kl_coef=0.1)
    need = lib.cm_token_workspace_bytes(rows, V)
    dx, o, a, lp, r, ww, st = torch.zeros(rows * V + 5 * rows + 8, device="cuda").split([rows * V] + 5 * [rows] + [8])  # dlogits as aligned as a tensor of its own: equal bits
    for dst, src in ((o, old), (a, adv), (r, ref), (ww, w)):
        dst.copy_(src)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    t = N.TokenRows(x.data_ptr(), V, None, 0, tok.data_ptr(), rows, V, N.DTYPE_F32, 8, 0, 1.0)
    N.check(lib.cm_token_policy_fwd_bwd(C.byref(t), o.data_ptr(), a.data_ptr(), r.data_ptr(), ww.data_ptr(), 0.2, 0.2, 0.1, 0.0, dx.data_ptr(), V, lp.data_ptr(), st.data_ptr(), ws.data_ptr(),
                                        need, N.raw_stream(0)), "cm_token_policy_fwd_bwd")
    assert torch.equal(lp, want.logp) and torch.equal(dx.view(rows, V), want.dlogits) and torch.equal(st, want.stats)


@pytest.mark.parametrize("keep", [torch.zeros(4, 2, dtype=torch.float16), torch.zeros(4, 2, dtype=torch.float64), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(2, 4).t(), torch.zeros(4), None])
def test_a_kept_softmax_of_another_type_is_refused(keep, monkeypatch):
    """token_logprob_bwd reads 8 bytes of `keep` for each row: fewer (16-bit values) would be read past its end."""
    from cleanmarl_amd import token_loss as TL
    monkeypatch.setattr(TL, "_rows", lambda *a: None)  # (the rows themselves would have to be on a GPU)
    row = torch.zeros(4)
    with pytest.raises(ValueError, match="keep=True"):
        TL.token_logprob_bwd(torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64), TL.TokenLogProb(row, None, keep), row)


def test_more_pairs_than_one_launch_has_workgroups_are_refused():
    """A launch ends at 2^32 threads, 2^24 workgroups of 256; a workgroup takes one pair."""
    from cleanmarl_amd import _native as N
    lib, t = N.load(), _rows()
    for pairs in (1 << 24, (1 << 31) - 1, 0, -1):
        assert lib.cm_preference_fwd_bwd(C.byref(t), 0x20000, pairs, 0x8000000, 0.1, 0.0, 0, 1.0, 0x30000, 8, None, None, 0x40000, 0x50000, 0, None) == -1
        assert "pairs=" in lib.cm_last_error().decode(), pairs
    assert lib.cm_preference_fwd_bwd(C.byref(t), 0x20000, (1 << 24) - 1, 0x8000000, 0.1, 0.0, 0, 1.0, 0x30000, 8, None, None, 0x40000, 0x50000, 0, None) == -1
    assert "workspace" in lib.cm_last_error().decode()


# ---------------------------------------------------------------------------------------------------------------- terms that are switched off
@pytest.mark.gpu
@pytest.mark.parametrize("V", [5, 700, 9000, 140003])
def test_a_reference_without_a_coefficient_only_measures(V):
    """kl_coef = 0 with logp_ref: the divergence is in the statistics and nowhere else, also where it is infinite (a row whose token is not available)."""
    from cleanmarl_amd import _native as N
    from cleanmarl_amd import token_loss as TL
    for dtype in (torch.float32, torch.bfloat16):
        x, tok, mask, gen = problem(6, V, dtype, V, avail=True)
        mask[0, tok[0]] = 0
        adv = torch.randn(6, generator=gen).cuda()
        old, ref = torch.full((6,), -2.0).cuda(), torch.full((6,), -2.5).cuda()
        for ent in (0.0, 0.01):
            a = TL.policy_loss_fwd_bwd(x, tok, old, adv, avail=mask, entropy_coef=ent)
            b = TL.policy_loss_fwd_bwd(x, tok, old, adv, logp_ref=ref, avail=mask, entropy_coef=ent)
            assert a.logp[0].item() == -math.inf and bool(torch.isfinite(a.dlogits).all())
            assert torch.equal(a.dlogits, b.dlogits) and torch.equal(a.logp, b.logp)
            keep = [i for i in range(8) if i != N.STAT_KL_REF]
            assert torch.equal(a.stats[keep].nan_to_num(7e37), b.stats[keep].nan_to_num(7e37)) and math.isfinite(b.stats[N.STAT_LOSS].item())
            assert a.stats[N.STAT_KL_REF].item() == 0.0 and b.stats[N.STAT_KL_REF].item() == math.inf
