"""Cases of the token-level training operators: log-probabilities, the clipped policy loss, the preference loss, AdamW over many tensors.

``run(state)`` computes one pass; with ``own`` false in elementary torch operations (32 bits inside, one rounding at the end), with ``own``
true through cleanmarl_amd.token_loss and cleanmarl_amd.adamw.  Both work on what ``prepare(case, seed)`` made.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
BLOCK = 256  # elements that share a scale in the 8-bit optimiser states; every tensor's states start at a multiple of it


def listed():
    return [
        # one new token of each of 16 sequences is scored: latency counts
        dict(name="logprob_single", op="logprob", rows=16, vocab=131072, dtype="bf16", entropy=0, grad=0, avail=0, temperature=1.0, ignore=0.0),
        # a batch of prompts scored by a frozen policy; odd vocabulary, so rows start at odd addresses; padding tokens are -100
        dict(name="logprob_prompt", op="logprob", rows=4096, vocab=50001, dtype="fp16", entropy=1, grad=0, avail=0, temperature=1.0, ignore=0.1),
        # log-probability and entropy of a caller's own loss, forward and backward, in 32 bits
        dict(name="logprob_grad", op="logprob", rows=2048, vocab=32000, dtype="fp32", entropy=1, grad=1, avail=0, temperature=0.8, ignore=0.0),
        # the action head of the 4096-env x 8-agent x 128-step workload: few actions, some unavailable, some rows with none
        dict(name="policy_agents", op="policy", rows=4194304, vocab=5, dtype="fp32", avail=1, temperature=1.0, kl=0.0, entropy=0.001, ignore=0.0),
        # a small minibatch of tokens: latency counts
        dict(name="policy_small", op="policy", rows=64, vocab=32768, dtype="bf16", avail=0, temperature=1.0, kl=0.05, entropy=0.0, ignore=0.0),
        # an ordinary minibatch of 8192 tokens over a large vocabulary
        dict(name="policy_tokens", op="policy", rows=8192, vocab=131072, dtype="bf16", avail=0, temperature=1.0, kl=0.05, entropy=0.0, ignore=0.0),
        # padded prompts and answers, odd vocabulary with forbidden tokens, sampled at a temperature, with an entropy bonus
        dict(name="policy_ragged", op="policy", rows=3001, vocab=100003, dtype="fp16", avail=1, temperature=0.7, kl=0.02, entropy=0.01, ignore=0.3),
        # eight pairs of long answers
        dict(name="preference_pairs", op="preference", pairs=8, longest=1024, ragged=0, vocab=65536, dtype="bf16", smoothing=0.0, kind="sigmoid", behind=0),
        # few short pairs of uneven lengths, packed, with unused rows behind the last one
        dict(name="preference_ragged", op="preference", pairs=5, longest=400, ragged=1, vocab=32001, dtype="fp32", smoothing=0.1, kind="sigmoid", behind=37),
        # the actor and the critic of the 4096-env workload in one step: small tensors, latency counts
        dict(name="adamw_agents", op="adamw", tensors=0, total=0, param="fp32", grad="fp32", copy=0, bits=32, clip=0.5),
        # a model of 268 million parameters: 32-bit masters, 16-bit gradients and a 16-bit copy for the next forward pass
        dict(name="adamw_model", op="adamw", tensors=120, total=268435456, param="fp32", grad="bf16", copy=1, bits=32, clip=1.0),
        # twice as many parameters in 16 bits with states in 8
        dict(name="adamw_8bit", op="adamw", tensors=200, total=536870912, param="bf16", grad="bf16", copy=0, bits=8, clip=0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprob", "policy", "preference", "adamw"])
    if op == "adamw":
        bits, total = rng.choice([8, 32]), _log_int(rng, 1 << 12, 1 << 27)
        param = rng.choice(["fp32", "bf16"])
        return dict(op=op, tensors=_log_int(rng, 1, 300), total=total, param=param, grad=rng.choice(["fp32", "bf16"]) if param == "fp32" else "bf16",
                    copy=rng.choice([0, 1]) if param == "fp32" else 0, bits=bits, clip=rng.choice([0.0, 1.0]) if bits == 32 else 0.0)
    vocab, dtype = _log_int(rng, 4, 131072), rng.choice(["fp32", "fp16", "bf16"])
    most = 1 << 27
    if op == "preference":
        pairs = _log_int(rng, 1, 16)
        return dict(op=op, pairs=pairs, longest=_log_int(rng, 1, max(1, min(1024, most // (2 * pairs * vocab)))), ragged=rng.choice([0, 1]), vocab=vocab,
                    dtype=dtype, smoothing=rng.choice([0.0, 0.1]), kind=rng.choice(["sigmoid", "sigmoid", "squared"]), behind=rng.choice([0, 13]))
    rows = _log_int(rng, 1, min(4194304 if op == "policy" else 65536, most // vocab))
    case = dict(op=op, rows=rows, vocab=vocab, dtype=dtype, avail=rng.choice([0, 1]), temperature=rng.choice([1.0, 0.7, 1.3]), ignore=rng.choice([0.0, 0.25]))
    if op == "logprob":
        return case | dict(entropy=rng.choice([0, 1]), grad=rng.choice([0, 1]))
    return case | dict(kl=rng.choice([0.0, 0.05]), entropy=rng.choice([0.0, 0.01]))


# ---------------------------------------------------------------------------------------------------------------- inputs
CLIP_LOW, CLIP_HIGH, BETA = 0.2, 0.2, 0.1
HYPER = dict(lr=3e-4, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1, step=7)


def _device():
    return torch.device("cuda")


def _logits(rows, vocab, dtype, gen, ignore):
    """Logits of a policy that is sure about some of its tokens, and the tokens it took (-100: none)."""
    dev = gen.device
    logits = torch.randn(rows, vocab, generator=gen, device=dev, dtype=dtype).mul_(2.0)
    token = torch.randint(vocab, (rows,), generator=gen, device=dev)
    sure = torch.rand(rows, generator=gen, device=dev).mul_(12.0).to(dtype)
    logits.scatter_add_(1, token[:, None], sure[:, None])
    if ignore:
        token = torch.where(torch.rand(rows, generator=gen, device=dev) < ignore, -100, token)
    return logits, token


def _avail(rows, vocab, token, gen):
    """Seven columns of ten available, the taken one always; one row of 64 has none."""
    dev = gen.device
    avail = (torch.rand(rows, vocab, generator=gen, device=dev, dtype=torch.float16) < 0.7).to(torch.uint8)
    avail.scatter_(1, token.clamp(min=0)[:, None], 1)
    avail[torch.randint(64, (rows,), generator=gen, device=dev) == 0] = 0
    return avail


def _taken(logits, token, avail, temperature):
    """log-probability of the taken tokens, in slices of rows."""
    got = []
    step = max(1, (1 << 27) // logits.shape[1])
    for i in range(0, logits.shape[0], step):
        x = logits[i:i + step].float() / temperature
        if avail is not None:
            x = torch.where(avail[i:i + step] != 0, x, -math.inf)
        got.append(torch.nan_to_num(x.gather(1, token[i:i + step].clamp(min=0)[:, None])[:, 0] - torch.logsumexp(x, 1), 0.0, 0.0, 0.0))
    return torch.cat(got)


def _off_the_border(noise):
    """Moves log ratios away from the two clip borders, next to which 32-bit rounding decides which branch a row takes."""
    for border in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
        noise = torch.where((noise - border).abs() < 1e-3, noise + 4e-3, noise)
    return noise


def _not_below_one_code(code):
    """The root of a second moment that is not zero keeps at least the smallest e4m3 value: a step never divides by a moment that was rounded away."""
    return torch.where((code > 0) & (code < 2.0 ** -9), 2.0 ** -9, code)


def _shapes(case):
    """Tensor sizes of an optimiser case: the two networks of the 4096-env workload, or a model's matrices, odd ones and vectors."""
    if case["tensors"] == 0:
        net = lambda din, dout: [64 * din, 64, 64 * 64, 64, 64 * dout, dout]  # noqa: E731
        return net(56, 5) + net(384, 1)
    rng = np.random.RandomState(case["tensors"])
    share = np.exp(rng.uniform(-4.0, 0.0, case["tensors"]))
    share[rng.rand(case["tensors"]) < 0.3] *= 1e-3
    return [max(1, int(n)) for n in share / share.sum() * case["total"]]


def prepare(case, seed):
    gen = torch.Generator(_device()).manual_seed(int(seed))
    dev = gen.device
    s = dict(case)
    if case["op"] == "adamw":
        sizes = _shapes(case)
        blocks = [-(-n // BLOCK) for n in sizes]
        total = sum(blocks) * BLOCK
        s["sizes"], s["starts"] = sizes, [BLOCK * b for b in np.cumsum([0] + blocks[:-1]).tolist()]
        real = torch.zeros(total, device=dev, dtype=torch.bool)
        for at, n in zip(s["starts"], sizes):
            real[at:at + n] = True

        def flat(scale, dtype):
            return torch.randn(total, generator=gen, device=dev, dtype=dtype).mul_(scale).mul_(real)

        s["param"] = flat(0.02, DTYPES[case["param"]])
        s["grad"] = flat(1e-3, DTYPES[case["grad"]])
        s["copy"] = s["param"].to(torch.bfloat16) if case["copy"] else None
        m = flat(5e-4, torch.float32)
        r = flat(1e-3, torch.float32).abs_()
        if case["bits"] == 32:
            s["exp_avg"], s["exp_avg_sq"] = m, r.square_()
        else:  # what a few steps leave behind: 8-bit codes and a scale for each block
            s["scale"] = torch.stack([m.view(-1, BLOCK).abs().amax(1), r.view(-1, BLOCK).amax(1)], 1) / 448.0
            s["exp_avg"] = (m.view(-1, BLOCK) / s["scale"][:, :1].clamp(min=1e-30)).to(torch.float8_e4m3fn).view(-1)
            s["root_avg_sq"] = _not_below_one_code(r.view(-1, BLOCK) / s["scale"][:, 1:].clamp(min=1e-30)).to(torch.float8_e4m3fn).view(-1)
        views = lambda t: None if t is None else [t[at:at + n] for at, n in zip(s["starts"], sizes)]  # noqa: E731
        s["params"], s["grads"], s["copies"] = views(s["param"]), views(s["grad"]), views(s["copy"])
        s["norm"] = torch.zeros(2, device=dev)
        if own:
            from cleanmarl_amd.adamw import MultiAdamW
            s["opt"] = MultiAdamW(s["params"], lr=HYPER["lr"], betas=(HYPER["beta1"], HYPER["beta2"]), eps=HYPER["eps"], weight_decay=HYPER["weight_decay"],
                                  state_bits=case["bits"], max_norm=case["clip"], copies=s["copies"])
            s["opt"].load_state(s["exp_avg"], s["exp_avg_sq"] if case["bits"] == 32 else s["root_avg_sq"], s.get("scale"), step=HYPER["step"] - 1)
        else:
            s["step"] = HYPER["step"] - 1
        return s
    if case["op"] == "preference":
        P, most = case["pairs"], case["longest"]
        rng = np.random.RandomState(1000 * P + most)  # the lengths belong to the case
        lengths = rng.randint(1, most + 1, 2 * P) if case["ragged"] else np.full(2 * P, most)
        start = np.concatenate([[0], np.cumsum(lengths)])
        rows = int(start[-1]) + case["behind"]
        s["logits"], s["token"] = _logits(rows, case["vocab"], DTYPES[case["dtype"]], gen, 0.2)
        s["seq_start"] = torch.tensor(start, dtype=torch.int32, device=dev)
        which = torch.repeat_interleave(torch.arange(2 * P, device=dev), torch.tensor(lengths, device=dev))
        logp = _taken(s["logits"], s["token"], None, 1.0)[:which.numel()] * (s["token"][:which.numel()] >= 0)
        total = torch.zeros(2 * P, device=dev, dtype=torch.float64).index_add_(0, which, logp.double())
        s["logp_ref"] = (total + 4.0 * torch.randn(2 * P, generator=gen, device=dev)).float()
        s["which"] = which
        s["dlogits"] = torch.zeros_like(s["logits"])
        return s
    s["logits"], s["token"] = _logits(case["rows"], case["vocab"], DTYPES[case["dtype"]], gen, case["ignore"])
    s["mask"] = _avail(case["rows"], case["vocab"], s["token"], gen) if case["avail"] else None
    if case["vocab"] <= 64:
        s["token"] = s["token"].to(torch.int32)
    randn = lambda: torch.randn(case["rows"], generator=gen, device=dev)  # noqa: E731
    s["adv"] = randn()
    if case["op"] == "logprob":
        s["d_logp"], s["d_entropy"] = s["adv"], randn().mul_(0.1)
    else:
        logp = _taken(s["logits"], s["token"].long(), s["mask"], case["temperature"])
        s["logp_old"] = logp - _off_the_border(randn().mul_(0.15))
        s["logp_ref"] = logp + randn().mul_(0.3) if case["kl"] else None
        s["weight"] = (torch.rand(case["rows"], generator=gen, device=dev) * 0.5 + 0.5)
    return s


# ---------------------------------------------------------------------------------------------------------------- the plain forms
def _plain_rows(logits, token, avail, temperature):
    """Parts of the softmax of each row that the formulas share."""
    x = logits.float()
    if avail is not None:
        x = torch.where(avail != 0, x, -math.inf)
    m = x.amax(1, keepdim=True)
    t = (x - torch.where(m == -math.inf, 0.0, m)) / temperature
    e = torch.exp(t)
    total = e.sum(1, keepdim=True)
    live = (token >= 0) & (total[:, 0] > 0)
    p = e / total
    log_sum = torch.log(total)
    at = token.clamp(min=0).long()[:, None]
    logp = torch.where(live, (t.gather(1, at) - log_sum)[:, 0], 0.0)
    return t, p, log_sum, at, logp, live


def _plain_entropy(t, p, log_sum, live, masked):
    pt = p * (torch.where(p > 0, t, 0.0) if masked else t)
    return torch.where(live, log_sum[:, 0] - pt.sum(1), 0.0)


def _plain_grad(g, h, t, p, log_sum, entropy, at, live, temperature, masked, dtype):
    """(g (1[token] - p) + h p (log p + H)) / T, zero in the rows left out."""
    d = -g[:, None] * p
    if h is not None:
        d = d + (h[:, None] * p) * ((torch.where(p > 0, t, 0.0) if masked else t) - log_sum + entropy[:, None])
    d.scatter_add_(1, at, g[:, None])
    return torch.where(live[:, None], d / temperature, 0.0).to(dtype)


def _plain_logprob(s):
    t, p, log_sum, at, logp, live = _plain_rows(s["logits"], s["token"], s["mask"], s["temperature"])
    out = {"logp": logp}
    masked = s["mask"] is not None
    if s["entropy"]:
        out["entropy"] = _plain_entropy(t, p, log_sum, live, masked)
    if s["grad"]:
        h = -s["d_entropy"] if s["entropy"] else None
        out["dlogits"] = _plain_grad(s["d_logp"], h, t, p, log_sum, out.get("entropy"), at, live, s["temperature"], masked, s["logits"].dtype)
    return out


def _plain_policy(s):
    t, p, log_sum, at, logp, live = _plain_rows(s["logits"], s["token"], s["mask"], s["temperature"])
    masked, c = s["mask"] is not None, s["entropy"]
    live = live & (s["weight"] != 0)
    H = _plain_entropy(t, p, log_sum, live, masked)
    ratio = torch.exp(logp - s["logp_old"])
    adv, w = s["adv"], torch.where(live, s["weight"], 0.0)
    whole, cut = adv * ratio, adv * ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
    pg = torch.minimum(whole, cut)
    g = torch.where(whole <= cut, -whole, 0.0)
    old_kl = (ratio - 1) - (logp - s["logp_old"])
    clipped = ((ratio < 1 - CLIP_LOW) | (ratio > 1 + CLIP_HIGH)).float()
    loss, kl = -pg - c * H, None
    if s["logp_ref"] is not None:
        d = s["logp_ref"] - logp
        kl = torch.expm1(d) - d
        g = g - s["kl"] * torch.expm1(d)
        loss = loss + s["kl"] * kl
    total = lambda v: torch.where(live, v * w, 0.0).double().sum()  # noqa: E731
    zero = torch.zeros((), device=w.device, dtype=torch.float64)
    stats = torch.stack([total(pg), total(H), total(old_kl), total(clipped), total(loss), live.double().sum(), zero if kl is None else total(kl), total(torch.ones_like(w))])
    dlogits = _plain_grad(w * g, w * c if c else None, t, p, log_sum, H, at, live, s["temperature"], masked, s["logits"].dtype)
    return {"stats": stats.float(), "logp": torch.where(live, logp, 0.0), "dlogits": dlogits}


def _plain_preference(s):
    which, P = s["which"], s["pairs"]
    n = which.numel()
    t, p, log_sum, at, logp, live = _plain_rows(s["logits"][:n], s["token"][:n], None, 1.0)
    L = torch.zeros(2 * P, device=logp.device, dtype=torch.float64).index_add_(0, which, logp.double())
    ratio = L - s["logp_ref"].double()
    margin = ratio[:P] - ratio[P:]
    if s["kind"] == "sigmoid":
        z, e = BETA * margin, s["smoothing"]
        softplus = lambda v: torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))  # noqa: E731
        loss = (1 - e) * softplus(-z) + e * softplus(z)
        d = BETA * (e / (1 + torch.exp(-z)) - (1 - e) / (1 + torch.exp(z)))
    else:
        d = 2 * (margin - 1 / (2 * BETA))
        loss = (margin - 1 / (2 * BETA)) ** 2
    stats = torch.stack([loss.sum(), (margin > 0).double().sum(), margin.sum(), L[:P].sum(), L[P:].sum(), torch.tensor(float(P), device=L.device, dtype=torch.float64)])
    g = (torch.cat([d, -d])[which] / P).float()
    s["dlogits"][:n] = _plain_grad(g, None, t, p, log_sum, None, at, live, 1.0, False, s["logits"].dtype)
    return {"stats": stats.float(), "margin": margin.float(), "seq_logp": L.float(), "dlogits": s["dlogits"]}


def _f32(x):
    return float(np.float32(x))


def _plain_adamw(s):
    s["step"] += 1
    h, bits = HYPER, s["bits"]
    g = s["grad"].float()
    if s["clip"]:
        norm = torch.sqrt(g.double().square().sum()).float()
        s["norm"][0] = norm
        g = g * torch.clamp(_f32(s["clip"]) / (norm + _f32(1e-6)), max=1.0)
    if bits == 32:
        m, v = s["exp_avg"], s["exp_avg_sq"]
    else:
        m = (s["exp_avg"].float().view(-1, BLOCK) * s["scale"][:, :1]).view(-1)
        v = (s["root_avg_sq"].float().view(-1, BLOCK) * s["scale"][:, 1:]).view(-1).square()
    m = m * _f32(h["beta1"]) + g * _f32(1 - h["beta1"])
    v = v * _f32(h["beta2"]) + (g * _f32(1 - h["beta2"])) * g
    root = torch.sqrt(v)
    denom = root * _f32(1 / math.sqrt(1 - h["beta2"] ** s["step"])) + _f32(h["eps"])
    p = s["param"].float() * _f32(1 - h["lr"] * h["weight_decay"]) - (m / denom) * _f32(h["lr"] / (1 - h["beta1"] ** s["step"]))
    s["param"].copy_(p)
    if s["copy"] is not None:
        s["copy"].copy_(p)
    if bits == 32:
        s["exp_avg"].copy_(m)
        s["exp_avg_sq"].copy_(v)
        return {"param": s["param"], "exp_avg": s["exp_avg"], "exp_avg_sq": s["exp_avg_sq"], "copy": s["copy"], "norm": s["norm"][0]}
    m, root = m.view(-1, BLOCK), root.view(-1, BLOCK)
    top = torch.stack([m.abs().amax(1), root.amax(1)], 1)
    scale = torch.where(top < 2.0 ** -100, 0.0, top * _f32(1 / 448))
    back = torch.where(scale > 0, 1.0 / scale, 0.0)
    s["exp_avg"].copy_((m * back[:, :1]).view(-1))
    s["root_avg_sq"].copy_(_not_below_one_code(root * back[:, 1:]).view(-1))
    s["scale"].copy_(scale)
    return {"param": s["param"], "exp_avg": s["exp_avg"], "root_avg_sq": s["root_avg_sq"], "scale": s["scale"]}


# ---------------------------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    if s["op"] == "adamw":
        opt = s["opt"]
        opt.step(s["grads"])
        if s["bits"] == 32:
            return {"param": s["param"], "exp_avg": opt.exp_avg, "exp_avg_sq": opt.exp_avg_sq, "copy": s["copy"], "norm": opt.norm[0] if s["clip"] else s["norm"][0]}
        return {"param": s["param"], "exp_avg": opt.exp_avg, "root_avg_sq": opt.root_avg_sq, "scale": opt.scale}
    from cleanmarl_amd import token_loss as TL
    if s["op"] == "logprob":
        r = TL.token_logprob(s["logits"], s["token"], avail=s["mask"], temperature=s["temperature"], entropy=bool(s["entropy"]), keep=bool(s["grad"]))
        out = {"logp": r.logp}
        if s["entropy"]:
            out["entropy"] = r.entropy
        if s["grad"]:
            out["dlogits"] = TL.token_logprob_bwd(s["logits"], s["token"], r, s["d_logp"], d_entropy=s["d_entropy"] if s["entropy"] else None,
                                                  avail=s["mask"], temperature=s["temperature"])
        return out
    if s["op"] == "policy":
        r = TL.policy_loss_fwd_bwd(s["logits"], s["token"], s["logp_old"], s["adv"], logp_ref=s["logp_ref"], weight=s["weight"], avail=s["mask"],
                                   temperature=s["temperature"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=s["kl"], entropy_coef=s["entropy"])
        return {"stats": r.stats, "logp": r.logp, "dlogits": r.dlogits}
    r = TL.preference_loss_fwd_bwd(s["logits"], s["token"], s["seq_start"], s["logp_ref"], beta=BETA, kind=s["kind"],
                                   label_smoothing=s["smoothing"] if s["kind"] == "sigmoid" else 0.0,  # the squared loss has none and refuses it
                                   scale=1.0 / s["pairs"], out=s["dlogits"])
    return {"stats": r.stats[:6], "margin": r.margin, "seq_logp": r.seq_logp, "dlogits": r.dlogits}


def run(s):
    if own:
        return _own(s)
    return {"logprob": _plain_logprob, "policy": _plain_policy, "preference": _plain_preference, "adamw": _plain_adamw}[s["op"]](s)


def work(case):
    if case["op"] == "adamw":
        sizes = _shapes(case)
        n, b = sum(sizes), 0
        b += 2 * BYTES[case["param"]] + BYTES[case["grad"]] + (2 if case["copy"] else 0)
        b += 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": n * b, "flops": n * (14 if case["bits"] == 32 else 22)}
    e = BYTES[case["dtype"]]
    if case["op"] == "preference":
        rows = 2 * case["pairs"] * ((case["longest"] + 1) / 2 if case["ragged"] else case["longest"])
        return {"bytes": rows * (2 * case["vocab"] * e + 8), "flops": rows * case["vocab"] * 8}
    # the rows left out are only written as zeros; what a mask leaves out of a row is read all the same
    rows, V, part = case["rows"], case["vocab"], 1 - case["ignore"]
    grad = case["op"] == "policy" or case["grad"]
    per_row = (32 if case["op"] == "policy" else 12) + (V * e if grad else 0) + part * V * (e + case["avail"])
    return {"bytes": rows * per_row, "flops": rows * part * V * (8 if grad else 4) + rows * V * (4 if case["entropy"] else 0)}


# ---------------------------------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_rows(x, token, avail, temperature):
    """x: 64-bit leaf.  (log-probability of the token, entropy, rows that count)."""
    z = x / temperature
    alive = token >= 0
    if avail is not None:
        alive = alive & (avail != 0).any(1)
        z = z.masked_fill((avail == 0) & alive[:, None], -1e5)  # e^-1e5 is 0 in 64 bits, and its product with -1e5 has a gradient
    lp = torch.log_softmax(z, 1)
    taken = lp[torch.arange(len(token), device=x.device), token.clamp(min=0).long()]
    return taken, -(lp.exp() * lp).sum(1), alive


def _exact_loss(s, taken, H, alive, a, b):
    """The scalar whose gradient a case returns, and its other outputs, for the rows [a, b)."""
    if s["op"] == "logprob":
        kept = torch.where(alive, taken, 0.0)
        loss = (kept * s["d_logp"][a:b].double()).sum()
        if s["entropy"]:
            loss = loss + (torch.where(alive, H, 0.0) * s["d_entropy"][a:b].double()).sum()
        return loss, None, kept, torch.where(alive, H, 0.0)
    alive = alive & (s["weight"][a:b] != 0)
    w, adv, old = (s[k][a:b].double() for k in ("weight", "adv", "logp_old"))
    delta = torch.where(alive, taken - old, 0.0)
    rho = delta.exp()
    pg = torch.minimum(adv * rho, adv * torch.clip(rho, 1 - CLIP_LOW, 1 + CLIP_HIGH))
    ent = torch.where(alive, H, 0.0)
    row = -pg - s["entropy"] * ent
    kl = torch.zeros_like(row)
    if s["logp_ref"] is not None:
        d = torch.where(alive, s["logp_ref"][a:b].double() - taken, 0.0)
        kl = d.exp() - 1 - d
        row = row + s["kl"] * kl
    w = torch.where(alive, w, 0.0)
    out = ((rho < 1 - CLIP_LOW) | (rho > 1 + CLIP_HIGH)).double()
    stats = torch.stack([(w * v).sum() for v in (pg, ent, rho - 1 - delta, out, row)] + [alive.double().sum(), (w * kl).sum(), w.sum()])
    return (w * row).sum(), stats, torch.where(alive, taken, 0.0), ent


def _exact_tokens(s):
    rows, V = s["logits"].shape
    step = max(1, (1 << 25) // V)
    grads, logps, ents, stats = [], [], [], 0
    for a in range(0, rows, step):
        b = min(rows, a + step)
        x = s["logits"][a:b].double().requires_grad_(True)
        mask = None if s["mask"] is None else s["mask"][a:b]
        taken, H, alive = _exact_rows(x, s["token"][a:b], mask, s["temperature"])
        wants_entropy = bool(s["entropy"])
        loss, st, logp, ent = _exact_loss(s, taken, H if wants_entropy else H.detach(), alive, a, b)
        if s["op"] == "policy" or s["grad"]:
            grads.append(torch.autograd.grad(loss, x)[0])
        logps.append(logp.detach())
        ents.append(ent.detach())
        stats = stats if st is None else stats + st.detach()
    out = {"logp": torch.cat(logps)}
    if s["op"] == "policy":
        return out | {"stats": stats, "dlogits": torch.cat(grads)}
    if s["entropy"]:
        out["entropy"] = torch.cat(ents)
    if s["grad"]:
        out["dlogits"] = torch.cat(grads)
    return out


def _exact_preference(s):
    P, start = s["pairs"], s["seq_start"].tolist()
    x_rows, L = s["logits"], []
    for q in range(2 * P):
        rows = slice(start[q], start[q + 1])
        z, tok = x_rows[rows].double(), s["token"][rows]
        L.append((torch.log_softmax(z, 1).gather(1, tok.clamp(min=0)[:, None])[:, 0] * (tok >= 0)).sum())
    L = torch.stack(L).requires_grad_(True)
    ratio = L - s["logp_ref"].double()
    margin = ratio[:P] - ratio[P:]
    if s["kind"] == "sigmoid":
        ls = torch.nn.functional.logsigmoid
        losses = -(1 - s["smoothing"]) * ls(BETA * margin) - s["smoothing"] * ls(-BETA * margin)
    else:
        losses = (margin - 0.5 / BETA) ** 2
    d = torch.autograd.grad(losses.mean(), L)[0].tolist()
    dlogits = torch.zeros(x_rows.shape, dtype=torch.float64, device=x_rows.device)
    for q in range(2 * P):
        rows = slice(start[q], start[q + 1])
        tok = s["token"][rows]
        dz = -torch.softmax(x_rows[rows].double(), 1)
        dz.scatter_add_(1, tok.clamp(min=0)[:, None], torch.ones_like(dz[:, :1]))
        dlogits[rows] = dz * (d[q] * (tok >= 0))[:, None]
    L, margin = L.detach(), margin.detach()
    stats = torch.stack([losses.detach().sum(), (margin > 0).sum().double(), margin.sum(), L[:P].sum(), L[P:].sum(), torch.full((), float(P), device=L.device, dtype=torch.float64)])
    return {"stats": stats, "margin": margin, "seq_logp": L, "dlogits": dlogits}


def _exact_adamw(s):
    h = HYPER
    g = s["grad"].double()
    norm = torch.zeros((), dtype=torch.float64, device=g.device)
    if s["clip"]:
        norm = g.norm()
        g = g * min(1.0, s["clip"] / (float(norm) + 1e-6))
    spread = lambda c: s["scale"][:, c].double().repeat_interleave(BLOCK)  # noqa: E731
    eight = s["bits"] == 8
    m = s["exp_avg"].float().double() * spread(0) if eight else s["exp_avg"].double()
    v = (s["root_avg_sq"].float().double() * spread(1)) ** 2 if eight else s["exp_avg_sq"].double()
    m = torch.lerp(m, g, 1 - h["beta1"])
    v = torch.addcmul(h["beta2"] * v, g, g, value=1 - h["beta2"])
    root = v.sqrt()
    m_hat, r_hat = m / (1 - h["beta1"] ** h["step"]), root / (1 - h["beta2"] ** h["step"]) ** 0.5
    p = s["param"].double() * (1 - h["lr"] * h["weight_decay"])
    p = torch.addcdiv(p, m_hat, r_hat + h["eps"], value=-h["lr"])
    if eight:  # the codes are whole steps apart: only the scales have a value in 64 bits
        scale = torch.stack([m.abs().view(-1, BLOCK).max(1).values, root.view(-1, BLOCK).max(1).values], 1) / 448
        return {"param": p, "exp_avg": None, "root_avg_sq": None, "scale": scale}
    return {"param": p, "exp_avg": m, "exp_avg_sq": v, "copy": p if s["copy"] is not None else None, "norm": norm}


def exact(case, seed):
    s = prepare(case, seed)
    return {"logprob": _exact_tokens, "policy": _exact_tokens, "preference": _exact_preference, "adamw": _exact_adamw}[case["op"]](s)
