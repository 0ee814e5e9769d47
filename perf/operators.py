"""Cases of the operators a policy with memory is trained and run with: layer
norm, the gated linear recurrence over a rollout's ticks (or any long
sequence), and the clipped policy loss with its KL term.

Sizes come from this repository's configurations -- 64 envs; 5,632 envs x 128
ticks with an MLP width of 128; 65,536 envs x 128 ticks in 8 minibatches; the
CNN's LN[16,13,13] .. LN[64,13,13]; heads of 5 moves and 2 bomb choices -- or
are generic long sequences and vocabularies, odd ones among them.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
CLIP_LOW, CLIP_HIGH, KL_COEF, ENT_COEF = 0.2, 0.28, 0.04, 0.01
_pkg = {}


def _ops():
    """The framework's operators (imported only where `own` is true)."""
    if not _pkg:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        path = os.path.join(root, "qqt-gpu-sim_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        from qqt_b200 import norm, policy_loss, recurrence
        _pkg.update(norm=norm, rec=recurrence, pl=policy_loss)
    return _pkg


def listed():
    ln, rec, pl = "layer_norm", "recurrence", "policy_loss"
    return [
        # one act() of 64 envs: the norm after the first layer, latency only
        dict(name="ln_act", op=ln, rows=64, d=128, pad=0, dtype="f32", train=False),
        # one tick of the CNN policy over 5,632 envs: its widest norm, LN[64,13,13]
        dict(name="ln_cnn_tick", op=ln, rows=5632, d=10816, pad=0, dtype="f16", train=False),
        # one minibatch of the large update: 65,536 envs x 128 ticks / 8 rows of width 128
        dict(name="ln_mlp_update", op=ln, rows=1048576, d=128, pad=0, dtype="f32", train=True),
        # a ragged minibatch of the CNN update, LN[16,13,13], its rows inside wider ones
        dict(name="ln_cnn_update", op=ln, rows=11267, d=2704, pad=24, dtype="bf16", train=True),
        # one tick of the memory over 5,632 envs (the rollout's form for single tokens)
        dict(name="rec_tick", op=rec, t=1, n=5632, d=128, batch_first=False, dtype="f32", mode="step"),
        # the update over one rollout: 128 ticks x 5,632 envs, episode ends inside
        dict(name="rec_rollout", op=rec, t=128, n=5632, d=128, batch_first=False, dtype="bf16",
             mode="train"),
        # one long sequence taken in at once: no parallelism but width and time
        dict(name="rec_long", op=rec, t=65536, n=1, d=1024, batch_first=True, dtype="bf16",
             mode="forward"),
        # a few long sequences of odd length and width, trained
        dict(name="rec_long_odd", op=rec, t=10007, n=3, d=517, batch_first=True, dtype="f32",
             mode="train"),
        # a small batch's loss: 64 envs x 4 ticks, both heads, latency only
        dict(name="loss_small", op=pl, rows=256, vocab=7, heads="5+2", legal=True, dtype="f32",
             mode="grad"),
        # one minibatch of the large update: both masked heads of 1,048,576 rows
        dict(name="loss_heads_update", op=pl, rows=1048576, vocab=7, heads="5+2", legal=True,
             dtype="f32", mode="grad"),
        # tokens of a language model's vocabulary: loss and gradient
        dict(name="loss_vocab", op=pl, rows=8192, vocab=32000, heads="", legal=False, dtype="bf16",
             mode="grad"),
        # log-probabilities and entropies of recorded tokens, a large odd vocabulary
        dict(name="score_vocab_odd", op=pl, rows=2047, vocab=100003, heads="", legal=False,
             dtype="f16", mode="score"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer_norm", "recurrence", "policy_loss"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    cells = _log(rng, 1 << 10, 1 << 25)            # values of the main input
    if op == "layer_norm":
        d = _log(rng, 16, 16384)
        return dict(op=op, rows=max(1, cells // d), d=d, pad=rng.choice([0, 0, 1, 8, 24]),
                    dtype=dtype, train=rng.random() < 0.6)
    if op == "recurrence":
        d = _log(rng, 16, 2048)
        mode = rng.choice(["step", "forward", "train", "train"])
        if mode == "step":
            return dict(op=op, t=1, n=max(1, cells // (16 * d)), d=d, batch_first=False, dtype=dtype,
                        mode=mode)
        t = _log(rng, 2, max(3, min(65536, cells // d)))
        return dict(op=op, t=t, n=max(1, cells // (d * t)), d=d, batch_first=rng.random() < 0.5,
                    dtype=dtype, mode=mode)
    mode = rng.choice(["grad", "grad", "score"])
    if rng.random() < 0.3:
        rows = max(1, cells // 32)
        return dict(op=op, rows=rows, vocab=7, heads="5+2", legal=True, dtype=dtype, mode=mode)
    vocab = _log(rng, 16, 150000)
    return dict(op=op, rows=max(1, 2 * cells // vocab), vocab=vocab, heads="",
                legal=rng.random() < 0.3, dtype=dtype, mode=mode)


def _segments(case):
    widths = [int(w) for w in case["heads"].split("+")] if case["heads"] else [case["vocab"]]
    at, out = 0, []
    for w in widths:
        out.append((at, at + w))
        at += w
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def rand(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    s = {"case": case}
    if case["op"] == "layer_norm":
        # pre-activations: every row has its own scale and offset
        n, d, w = case["rows"], case["d"], case["d"] + case["pad"]
        s["x"] = (randn(n, w) * (0.5 + rand(n, 1)) + 0.5 * randn(n, 1)).to(dt)[:, :d]
        s["w"] = 1 + 0.1 * randn(d)
        s["b"] = 0.1 * randn(d)
        if case["train"]:
            s["dy"] = randn(n, d).to(dt)
        return s
    if case["op"] == "recurrence":
        t, n, d = case["t"], case["n"], case["d"]
        first, second = (n, t) if case["batch_first"] else (t, n)

        def seq(v):
            return v.transpose(0, 1) if case["batch_first"] else v

        # candidate and gate come out of one linear layer, side by side
        both = randn(first, second, 2 * d)
        both[..., d:] = both[..., d:] * 1.5 + 2.0      # gates that mostly remember
        both = both.to(dt)
        s["x"], s["gate"] = seq(both[..., :d]), seq(both[..., d:])
        s["reset"] = rand(t, n) < 1.0 / 80             # an episode's first tick
        s["h0"] = randn(n, d)
        if case["mode"] == "step":
            s["x"], s["gate"], s["reset"] = s["x"][0], s["gate"][0], s["reset"][0]
        if case["mode"] == "train":
            s["dh"] = seq(randn(first, second, d).to(dt))
            s["dh_last"] = randn(n, d)
        return s
    n, v = case["rows"], case["vocab"]
    logits = (2.5 * randn(n, v)).to(dt)
    segs = _segments(case)
    legal = None
    if case["legal"]:
        legal = rand(n, v) < 0.6
        legal[:, [a for a, _ in segs]] = True          # the first choice (stay, no bomb) always is
    z = logits.float() if legal is None else logits.float().masked_fill(~legal, -math.inf)
    noise = z - torch.log(-torch.log(rand(n, v).clamp(1e-7, 1 - 1e-6)))
    acts, logp = [], 0
    for a, b in segs:
        pick = noise[:, a:b].argmax(1)
        acts.append(pick)
        lp = z[:, a:b].gather(1, pick[:, None])[:, 0] - z[:, a:b].logsumexp(1)
        logp = logp + lp
    s["logits"], s["legal"] = logits, legal
    s["actions"] = torch.stack(acts, 1)
    if case["mode"] == "grad":
        # most tokens close to the policy that drew them, one in twenty far from it; the
        # ratios stay off the clip's two edges, where the loss has two one-sided slopes
        far = (0.3 + 0.5 * rand(n)) * torch.sign(rand(n) - 0.5)
        s["old_logp"] = logp - torch.where(rand(n) < 0.05, far, 0.04 * randn(n))
        s["ref_logp"] = logp + 0.3 * randn(n)
        s["adv"] = randn(n)
        s["mask"] = rand(n) < 0.9                      # padding and frames that do not count
        # half-precision gradients of a mean over n rows are scaled, as mixed-precision
        # training does
        s["grad_scale"] = 64.0 * n if case["dtype"] == "f16" else 1.0
    s["heads"] = [b - a for a, b in segs]
    return s


def _scan(a, b, h0):
    """h_t = a_t h_{t-1} + b_t over dim 0 by doubling: every round composes each
    step with the one `k` earlier."""
    a, b = a.clone(), b.clone()
    b[0] += a[0] * h0
    k, t = 1, a.shape[0]
    while k < t:
        b = torch.cat([b[:k], b[k:] + a[k:] * b[:-k]])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return b


def _plain_layer_norm(s):
    x, w = s["x"].float(), s["w"]
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + EPS)
    xh = c * rstd
    out = {"y": (xh * w + s["b"]).to(s["x"].dtype)}
    if s["case"]["train"]:
        dy = s["dy"].float()
        gw = dy * w
        dx = rstd * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
        out.update(dx=dx.to(s["x"].dtype), dw=(dy * xh).sum(0), db=dy.sum(0))
    return out


def _plain_recurrence(s):
    mode, dt = s["case"]["mode"], s["x"].dtype
    x, g = s["x"].float(), s["gate"].float()
    keep = (~s["reset"]).float()[..., None]
    f = torch.sigmoid(g)
    i = torch.sigmoid(-g)
    if mode == "step":
        h = f * keep * s["h0"] + i * x
        return {"h": h.to(dt), "state": h}
    a = f * keep
    h = _scan(a, i * x, s["h0"])
    out = {"h": h.to(dt), "h_last": h[-1]}
    if mode == "train":
        dy = s["dh"].float()
        # the same scan backwards in time: step t is fed by step t + 1 through a_{t+1}
        a_next = torch.cat([a[1:], torch.ones_like(a[:1])]).flip(0)
        d = _scan(a_next, dy.flip(0), s["dh_last"]).flip(0)
        prev = torch.cat([s["h0"][None], h[:-1]])
        out.update(dx=(i * d).to(dt), dgate=(f * i * d * (keep * prev - x)).to(dt), dh0=a[0] * d[0])
    return out


def _plain_policy(s):
    logits, legal = s["logits"], s["legal"]
    z = logits.float() if legal is None else logits.float().masked_fill(~legal, -math.inf)
    parts, logp, ent = [], 0, 0
    for a, b, k in _spans(s):
        zz = z[:, a:b]
        c = zz - zz.amax(1, keepdim=True)
        e = c.exp()
        total = e.sum(1, keepdim=True)
        lp = c - total.log()
        p = e / total
        h = -(p * torch.where(p > 0, lp, 0)).sum(1, keepdim=True)
        act = s["actions"][:, k:k + 1]
        logp = logp + lp.gather(1, act)[:, 0]
        ent = ent + h[:, 0]
        parts.append((p, lp, h, act))
    if s["case"]["mode"] == "score":
        return {"logp": logp, "entropy": ent}
    adv, mask = s["adv"], s["mask"].float()
    count = mask.sum().clamp(min=1)
    ratio = (logp - s["old_logp"]).exp()
    clipped = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
    pg = -torch.minimum(ratio * adv, clipped * adv)
    delta = s["ref_logp"] - logp
    kl = torch.expm1(delta) - delta
    outside = ((ratio < 1 - CLIP_LOW) | (ratio > 1 + CLIP_HIGH)).float()
    pg, kl, h, cf = ((v * mask).sum() / count for v in (pg, kl, ent, outside))
    stats = torch.stack([pg + KL_COEF * kl - ENT_COEF * h, pg, kl, h, cf])
    live = ~(((adv > 0) & (ratio > 1 + CLIP_HIGH)) | ((adv < 0) & (ratio < 1 - CLIP_LOW)))
    scale = mask * s["grad_scale"] / count
    coef = ((-adv * ratio * live - KL_COEF * torch.expm1(delta)) * scale)[:, None]
    ec = (ENT_COEF * scale)[:, None]
    grads = []
    for p, lp, h, act in parts:
        dz = -coef * p + ec * p * torch.where(p > 0, lp + h, 0)
        grads.append(dz.scatter_add(1, act, coef))
    return {"stats": stats, "logp": logp, "dlogits": torch.cat(grads, 1).to(logits.dtype)}


def _spans(s):
    ends = [sum(s["heads"][:k + 1]) for k in range(len(s["heads"]))]
    return [(e - w, e, k) for k, (e, w) in enumerate(zip(ends, s["heads"]))]


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"layer_norm": _plain_layer_norm, "recurrence": _plain_recurrence,
                "policy_loss": _plain_policy}[op](s)
    k = _ops()
    if op == "layer_norm":
        if not s["case"]["train"]:
            return {"y": k["norm"].layer_norm(s["x"], s["w"], s["b"], EPS)}
        y, mean, rstd = k["norm"].layer_norm_forward(s["x"], s["w"], s["b"], EPS)
        dx, dw, db = k["norm"].layer_norm_backward(s["dy"], s["x"], mean, rstd, s["w"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if op == "recurrence":
        rec, mode = k["rec"], s["case"]["mode"]
        if mode == "step":
            h, state = rec.gated_recurrence_step(s["x"], s["gate"], s["h0"], s["reset"])
            return {"h": h, "state": state}
        if mode == "forward":
            h, last = rec.gated_recurrence(s["x"], s["gate"], s["h0"], s["reset"])
            return {"h": h, "h_last": last}
        h, last, saved = rec.gated_recurrence_forward(s["x"], s["gate"], s["h0"], s["reset"])
        dx, dg, dh0 = rec.gated_recurrence_backward(s["dh"], s["dh_last"], s["x"], s["gate"], saved,
                                                    s["reset"])
        return {"h": h, "h_last": last, "dx": dx, "dgate": dg, "dh0": dh0}
    if s["case"]["mode"] == "score":
        logp, ent = k["pl"].policy_logp(s["logits"], s["actions"], legal=s["legal"],
                                        heads=s["heads"])
        return {"logp": logp, "entropy": ent}
    stats, logp, dz = k["pl"].policy_loss_and_grad(
        s["logits"], s["actions"], s["old_logp"], s["adv"], ref_logp=s["ref_logp"],
        legal=s["legal"], mask=s["mask"], heads=s["heads"], clip=(CLIP_LOW, CLIP_HIGH),
        kl_coef=KL_COEF, entropy_coef=ENT_COEF, grad_scale=s["grad_scale"])
    return {"stats": stats, "logp": logp, "dlogits": dz}


def work(case):
    u = SIZE[case["dtype"]]
    if case["op"] == "layer_norm":
        n, d = case["rows"], case["d"]
        if not case["train"]:
            return {"bytes": 2 * u * n * d + 8 * d, "flops": 8 * n * d}
        return {"bytes": 4 * u * n * d + 16 * d, "flops": 22 * n * d}
    if case["op"] == "recurrence":
        c, nd = case["t"] * case["n"] * case["d"], case["n"] * case["d"]
        flags = case["t"] * case["n"]
        if case["mode"] == "train":       # x, gate, dh -> h, dx, dgate; h0, dh_last -> h_last, dh0
            return {"bytes": 6 * u * c + 16 * nd + flags, "flops": 24 * c}
        return {"bytes": 3 * u * c + 8 * nd + flags, "flops": 8 * c}
    n, v = case["rows"], case["vocab"]
    nh = len(_segments(case))
    legal = n * v if case["legal"] else 0
    if case["mode"] == "score":
        return {"bytes": u * n * v + legal + 8 * n * nh + 8 * n, "flops": 6 * n * v}
    return {"bytes": 2 * u * n * v + legal + 8 * n * nh + 4 * 4 * n + n, "flops": 14 * n * v}


def exact(case, seed):
    """The definitions in 64 bits: the norm by its variance and its Jacobian, the
    recurrence tick by tick, the loss through automatic differentiation."""
    s = prepare(case, seed)
    if case["op"] == "layer_norm":
        x, w = s["x"].double(), s["w"].double()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        xh = (x - mean) / (var + EPS).sqrt()
        out = {"y": xh * w + s["b"].double()}
        if case["train"]:
            q = s["dy"].double()
            out["dw"], out["db"] = torch.einsum("nd,nd->d", q, xh), q.sum(0)
            q = q * w
            # (I - 1 1'/d - xh xh'/d) q, by rows
            q = q - q.mean(1, keepdim=True) - xh * torch.einsum("nd,nd->n", q, xh)[:, None] / case["d"]
            out["dx"] = q / (var + EPS).sqrt()
        return out
    if case["op"] == "recurrence":
        dd = torch.float64
        one_tick = case["mode"] == "step"
        x, g, r = ((v[None] if one_tick else v) for v in (s["x"], s["gate"], s["reset"]))
        x, g = x.to(dd).contiguous(), g.to(dd).contiguous()
        f = 1 / (1 + torch.exp(-g))
        hs = torch.empty_like(x)
        before = torch.empty_like(x)
        h = s["h0"].to(dd)
        keep = (~r).to(dd)[..., None]
        for t in range(x.shape[0]):
            before[t] = keep[t] * h
            h = x[t] + f[t] * (before[t] - x[t])
            hs[t] = h
        if one_tick:
            return {"h": hs[0], "state": hs[0]}
        out = {"h": hs, "h_last": hs[-1]}
        if case["mode"] == "train":
            d = s["dh_last"].to(dd)
            dx, dgate = torch.empty_like(x), torch.empty_like(x)
            dh = s["dh"].to(dd).contiguous()
            for t in reversed(range(x.shape[0])):
                d = d + dh[t]
                dx[t] = d * (1 - f[t])
                dgate[t] = d * (before[t] - x[t]) * f[t] * (1 - f[t])
                d = d * f[t] * keep[t]
            out.update(dx=dx, dgate=dgate, dh0=d)
        return out
    z = s["logits"].double()
    if s["legal"] is not None:
        z = torch.where(s["legal"], z, torch.full((), -1e300, device=z.device, dtype=z.dtype))
    z.requires_grad_(case["mode"] == "grad")
    logp, ent = 0, 0
    for k, part in enumerate(torch.split(z, s["heads"], 1)):
        lp = torch.log_softmax(part, 1)
        logp = logp + lp.gather(1, s["actions"][:, k:k + 1])[:, 0]
        ent = ent - (lp.exp() * lp).sum(1)
    if case["mode"] == "score":
        return {"logp": logp, "entropy": ent}
    m = s["mask"].double() / max(1, int(s["mask"].sum()))
    ratio = torch.exp(logp - s["old_logp"].double())
    adv = s["adv"].double()
    pg = -torch.minimum(ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv)
    diff = s["ref_logp"].double() - logp
    kl = torch.expm1(diff) - diff
    far = ((ratio - 1 > CLIP_HIGH) | (1 - ratio > CLIP_LOW)).double()
    pg, kl, h, far = (torch.dot(v, m) for v in (pg, kl, ent, far))
    loss = pg + KL_COEF * kl - ENT_COEF * h
    grad, = torch.autograd.grad(loss * s["grad_scale"], z)
    return {"stats": torch.stack([loss, pg, kl, h, far]).detach(), "logp": logp.detach(),
            "dlogits": grad}
