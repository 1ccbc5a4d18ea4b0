"""What is measured of the objectives over a model's logits: token
log-probabilities, the clipped policy loss, the preference loss and the
distillation loss of `dop.losses`, each beside its plain form in elementary
torch operations."""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}


# ------------------------------------------------------------------- cases
def listed():
    """V 32000 is the vocabulary of the Mixtral configuration; 32768 rows are
    the Mixtral block workload's 8 sequences of 4096 tokens."""
    return [
        # the log-probability of a few sampled tokens: latency
        _case("logp_small", "logp", rows=4, vocab=32000, type="f32"),
        # a frozen reference policy's scoring pass over four sequences, prompts masked
        _case("logp_reference", "logp", rows=16384, vocab=32000, type="bf16", masked=0.2),
        # an objective of the user's own: its dlogp taken back to the logits; odd vocabulary
        _case("logp_backward", "logp_backward", rows=4095, vocab=50001, type="f32", grad="bf16"),
        # one short rollout in the fp32 model
        _case("policy_small", "policy", rows=61, vocab=32000, type="f32", grad="f32", kl=0.05),
        # a batch of rollouts in the bf16 model (fp32 logits, bf16 cotangent), prompts masked
        _case("policy_rollouts", "policy", rows=8192, vocab=32000, type="f32", grad="bf16",
              masked=0.25, kl=0.05, tau=0.8),
        # a large odd vocabulary: no row starts on a 16-byte boundary
        _case("policy_odd_vocab", "policy", rows=3001, vocab=100003, type="bf16", grad="bf16"),
        # two short preference pairs: latency
        _case("preference_small", "preference", rows=48, vocab=32000, type="f32", grad="f32",
              pairs=2),
        # a batch of ragged pairs of about 512 tokens a sequence, prompts masked
        _case("preference_batch", "preference", rows=16384, vocab=32000, type="bf16", grad="bf16",
              pairs=16, masked=0.3),
        # the smallest distillation call
        _case("distill_small", "distill", rows=16, vocab=32000, type="f32", grad="f32", top=32),
        # the whole batch of the Mixtral block workload, 64 teacher logits a token
        _case("distill_batch", "distill", rows=32768, vocab=32000, type="bf16", grad="bf16",
              top=64, tau=2.0),
        # a large vocabulary with the teacher's remaining mass as one more class
        _case("distill_tail", "distill", rows=2047, vocab=128000, type="f32", grad="f32", top=128,
              tail=True),
        # odd vocabulary inside padded rows, fp32 logits to a bf16 cotangent
        _case("distill_padded", "distill", rows=5000, vocab=32003, pad=13, type="f32",
              grad="bf16", top=20, tail=True, masked=0.1),
    ]


def _case(name, op, rows, vocab, type, grad="", pad=0, masked=0.0, tau=1.0, kl=0.0, pairs=0,
          top=0, tail=False):
    c = {"op": op, "rows": rows, "vocab": vocab, "type": type, "grad": grad, "pad": pad,
         "masked": masked, "tau": tau, "kl": kl, "pairs": pairs, "top": top, "tail": tail}
    return {"name": name, **c} if name else c


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logp", "logp_backward", "policy", "preference", "distill"])
    vocab = _log_uniform(rng, 32, 160000)
    if rng.random() < 0.5:
        vocab += vocab % 2 + 1  # odd
    rows = _log_uniform(rng, 1, max(1, min(16384, 400_000_000 // vocab)))
    type, grad = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
    pad = rng.choice([0, 0, 0, rng.randint(1, 64)])
    masked = rng.choice([0.0, round(rng.uniform(0.05, 0.6), 2)])
    tau = rng.choice([1.0, round(rng.uniform(0.5, 3.0), 2)])
    pairs = top = 0
    kl, tail = 0.0, False
    if op == "policy":
        kl = rng.choice([0.0, round(rng.uniform(0.01, 0.2), 3)])
    if op == "preference":
        rows = max(rows, 4)
        pairs = _log_uniform(rng, 1, max(1, min(rows // 4, 64)))
    if op == "distill":
        top = _log_uniform(rng, 1, min(256, vocab // 2))
        tail = rng.random() < 0.5
    if op == "logp":
        grad = ""
    return _case("", op, rows, vocab, type, grad, pad, masked, tau, kl, pairs, top, tail)


def _masked(case):
    return int(case["masked"] * case["rows"])


def _sequences(case):
    """Row offsets of the 2 * pairs sequences, and each sequence's masked
    prompt rows: ragged, from the case alone.  A few rows stay behind the
    last sequence."""
    rng = random.Random(case["rows"] * 1009 + case["pairs"])
    n, rows = 2 * case["pairs"], case["rows"]
    used = rows - min(rows - n, rows // 50)
    share = [rng.uniform(0.4, 1.6) for _ in range(n)]
    total, at, off = sum(share), 0.0, [0]
    for i, s in enumerate(share):
        at += s / total * (used - n)
        off.append(int(at) + i + 1)
    off[-1] = used
    prompt = [int(case["masked"] * (b - a)) for a, b in zip(off, off[1:])]
    return off, prompt


def _active(case):
    """Rows whose logits count."""
    if case["op"] == "preference":
        off, prompt = _sequences(case)
        return off[-1] - sum(prompt)
    return case["rows"] - _masked(case)


def work(case):
    T, V, A = case["rows"], case["vocab"], _active(case)
    read = A * V * BYTES[case["type"]] + 12 * T  # logits, tokens, weights
    write = T * V * BYTES[case["grad"]] if case["grad"] else 0
    # an element's part in the softmax: scale, subtract, exponential, add; in
    # the gradient: subtract, exponential, multiply
    flops = A * V * {"logp": 4, "logp_backward": 4}.get(case["op"], 7)
    if case["op"] in ("logp", "logp_backward"):
        read += 0 if case["op"] == "logp" else 8 * T
        write += 8 * T if case["op"] == "logp" else 0
    elif case["op"] == "policy":
        read += 12 * T
        write += 8 * T
    elif case["op"] == "preference":
        read += 4 * T
        write += 4 * T
    else:
        read += (8 * case["top"] + 4 * case["tail"] - 8) * T
        write += 4 * T
    return {"bytes": read + write, "flops": flops}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, V, tau = case["rows"], case["vocab"], case["tau"]

    def normal(*n):
        return torch.randn(*n, generator=g, device="cuda")

    def whole(hi, *n):
        return torch.randint(0, hi, n, generator=g, device="cuda")

    buf = torch.empty(T, V + case["pad"], dtype=TYPES[case["type"]], device="cuda")
    buf.normal_(0.0, 2.5, generator=g)
    z = buf[:, :V]
    tokens = whole(V, T)
    # the token a policy has sampled is one that it finds likely
    rows = torch.arange(T, device="cuda")
    z[rows, tokens] += 6.0
    weight = torch.ones(T, device="cuda")
    s = {"case": case, "z": z, "tokens": tokens, "weight": weight,
         "scale": 1.0 / max(1, _active(case))}
    if case["op"] != "preference":
        weight[torch.randperm(T, generator=g, device="cuda")[:_masked(case)]] = 0.0
    if case["op"] == "distill":
        # the teacher's logits: near the student's on some entries, its own on others
        K = case["top"]
        index = torch.argsort(torch.rand(min(T, 64), V, generator=g, device="cuda"), 1)[:, :K]
        shift = whole(V, T, 1)
        index = (index[rows % index.shape[0]] + shift) % V  # distinct in a row
        index[:, 0] = torch.where((index == tokens[:, None]).any(1), index[:, 0], tokens)
        y = z.gather(1, index).float() * 0.7 + 3.0 * normal(T, K) + 2.0
        y, order = y.sort(1, descending=True)
        s["top_index"] = index.gather(1, order).int().contiguous()
        s["top_logit"] = y.contiguous()
        s["teacher_lse"] = None
        if case["tail"]:  # between 2% and 40% of the teacher's mass lies outside the K
            out = 0.02 + 0.38 * torch.rand(T, generator=g, device="cuda")
            s["teacher_lse"] = torch.logsumexp(y / tau, 1) - torch.log1p(-out)
        return s
    if case["op"] == "logp":
        return s
    lse = torch.cat([torch.logsumexp(c.double() / tau, 1) for c in z.split(512)])
    logp = (z[rows, tokens].double() / tau - lse).float()
    if case["op"] == "logp_backward":
        s["lse"] = lse.float()
        s["dlogp"] = normal(T) * s["scale"] * weight
        return s
    s["ref_logp"] = logp + 0.3 * normal(T)
    if case["op"] == "policy":
        # the policy has moved a little since the rollout, mostly where the
        # advantage pointed; no ratio lies within
        # 1e-3 of a border of the clip, where the last bit of a 32-bit log
        # probability would decide the branch
        s["advantage"] = normal(T)
        moved = 0.2 * s["advantage"] + 0.15 * normal(T)
        for border in (math.log(1.0 - CLIP_LOW), math.log(1.0 + CLIP_HIGH)):
            near = (moved - border).abs() < 1e-3
            moved = torch.where(near, moved + 4e-3, moved)
        s["old_logp"] = logp - moved
        if not case["kl"]:
            s["ref_logp"] = None
    else:
        off, prompt = _sequences(case)
        s["seq_off"] = off
        for a, n in zip(off, prompt):
            weight[a:a + n] = 0.0
        s["scale"] = 1.0 / case["pairs"]
    return s


CLIP_LOW, CLIP_HIGH = 0.2, 0.28
BETA, SMOOTHING = 0.1, 0.05


# ------------------------------------------------------------- plain forms
def run(s):
    return _own(s) if own else PLAIN[s["case"]["op"]](s)


def _softmax(s):
    """x = z / tau and softmax(x) in 32 bits, log sum exp x in 64 from the
    32-bit sum: ratios and margins are small differences of log-probabilities."""
    x = s["z"].float() / s["case"]["tau"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    t = e.sum(1, keepdim=True)
    return x, m[:, 0].double() + torch.log(t[:, 0].double()), e / t


def _onehot_minus(p, tokens, c):
    """c [T] times (one at the token minus p), in place of p."""
    d = p * -c[:, None]
    rows = torch.arange(p.shape[0], device=p.device)
    d[rows, tokens] += c
    return d


def _plain_logp(s):
    x, tokens, weight = s["z"].float() / s["case"]["tau"], s["tokens"], s["weight"]
    m = x.amax(1, keepdim=True)
    lse = m[:, 0] + torch.log(torch.exp(x - m).sum(1))
    logp = x.gather(1, tokens[:, None])[:, 0] - lse
    zero = torch.zeros_like(lse)
    return {"logp": torch.where(weight != 0, logp, zero), "lse": torch.where(weight != 0, lse, zero)}


def _plain_logp_backward(s):
    x = s["z"].float() / s["case"]["tau"]
    p = torch.exp(x - s["lse"][:, None])
    d = _onehot_minus(p, s["tokens"], s["dlogp"] / s["case"]["tau"])
    return {"dlogits": d.to(TYPES[s["case"]["grad"]])}


def _plain_policy(s):
    case, w = s["case"], s["weight"]
    x, lse, p = _softmax(s)
    logp = x.gather(1, s["tokens"][:, None])[:, 0] - lse
    A = s["advantage"]
    r = torch.exp(logp - s["old_logp"])
    clipped = ((A > 0) & (r > 1 + CLIP_HIGH)) | ((A < 0) & (r < 1 - CLIP_LOW))
    l = -torch.minimum(r * A, r.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * A)
    d = torch.where(clipped, torch.zeros_like(r), -A * r)
    if s["ref_logp"] is not None:
        gap = s["ref_logp"] - logp
        l = l + case["kl"] * (torch.expm1(gap) - gap)
        d = d - case["kl"] * torch.expm1(gap)
    l = w * l
    dz = _onehot_minus(p, s["tokens"], (s["scale"] * w * d / case["tau"]).float())
    return {"loss": (s["scale"] * l.sum()).float(), "row_loss": l.float(),
            "logp": torch.where(w != 0, logp, torch.zeros_like(logp)).float(),
            "dlogits": dz.to(TYPES[case["grad"]])}


def _plain_preference(s):
    case, w = s["case"], s["weight"]
    x, lse, p = _softmax(s)
    logp = x.gather(1, s["tokens"][:, None])[:, 0] - lse
    off = torch.tensor(s["seq_off"], device=w.device)
    rows = torch.arange(w.shape[0], device=w.device)
    seq = torch.bucketize(rows, off, right=True) - 1  # 2 * pairs: behind the last sequence
    inside = rows < off[-1]
    run_ = torch.cumsum(w * (logp - s["ref_logp"]), 0)
    run_ = torch.cat([run_.new_zeros(1), run_])
    sums = run_[off[1:]] - run_[off[:-1]]
    m = BETA * (sums[0::2] - sums[1::2])

    def minus_log_sigma(v):
        return torch.clamp(-v, min=0) + torch.log1p(torch.exp(-v.abs()))

    l = (1 - SMOOTHING) * minus_log_sigma(m) + SMOOTHING * minus_log_sigma(-m)
    dm = -(1 - SMOOTHING) / (1 + torch.exp(m)) + SMOOTHING / (1 + torch.exp(-m))
    c = torch.stack([dm, -dm], 1).reshape(-1) * (BETA * s["scale"])
    c = torch.cat([c, c.new_zeros(1)])[seq].float() * w * inside
    dz = _onehot_minus(p, s["tokens"], c / case["tau"])
    return {"loss": (s["scale"] * l.sum()).float(), "pair_loss": l.float(), "margin": m.float(),
            "logp": torch.where(inside & (w != 0), logp, torch.zeros_like(logp)).float(),
            "dlogits": dz.to(TYPES[case["grad"]])}


def _plain_distill(s):
    case, w, tau = s["case"], s["weight"], s["case"]["tau"]
    index = s["top_index"].long()
    x, lse, p = _softmax(s)
    logp = x.gather(1, index) - lse[:, None]
    y = s["top_logit"] / tau
    if s["teacher_lse"] is None:
        m = y.amax(1, keepdim=True)
        logq = y - m - torch.log(torch.exp(y - m).sum(1, keepdim=True))
        q = torch.exp(logq)
        l = (q * (logq - logp)).sum(1)
        d = p
    else:
        logq = y - s["teacher_lse"][:, None]
        q = torch.exp(logq)
        qr = (1 - q.sum(1)).clamp(min=0)
        # the student's mass outside the K entries, summed there
        rest = p.clone()
        rest.scatter_(1, index, 0.0)
        pr = rest.sum(1)
        some = torch.where(qr > 0, qr, torch.ones_like(qr))
        l = (q * (logq - logp)).sum(1) + qr * (torch.log(some) - torch.log(pr))
        d = p - rest * (qr / pr)[:, None]
    d.scatter_add_(1, index, -q)
    l = w * (tau * tau) * l
    d *= (s["scale"] * tau * w)[:, None]
    return {"loss": (s["scale"] * l.sum()).float(), "row_loss": l.float(),
            "dlogits": d.to(TYPES[case["grad"]])}


PLAIN = {"logp": _plain_logp, "logp_backward": _plain_logp_backward, "policy": _plain_policy,
         "preference": _plain_preference, "distill": _plain_distill}


# --------------------------------------------------- the framework's calls
def _losses():
    if "dop" not in sys.modules:
        sys.path.insert(0, os.path.join(ROOT, "dependent-optics_b200"))
    from dop import losses
    return losses


def _own(s):
    losses, case = _losses(), s["case"]
    tau, op = case["tau"], case["op"]
    grad = TYPES.get(case["grad"])
    if op == "logp":
        logp, lse = losses.token_logp(s["z"], s["tokens"], weight=s["weight"], temperature=tau)
        return {"logp": logp, "lse": lse}
    if op == "logp_backward":
        d = losses.token_logp_backward(s["z"], s["tokens"], s["lse"], s["dlogp"], temperature=tau,
                                       grad_dtype=grad)
        return {"dlogits": d}
    if op == "policy":
        r = losses.policy_loss(s["z"], s["tokens"], s["old_logp"], s["advantage"],
                               ref_logp=s["ref_logp"], weight=s["weight"], temperature=tau,
                               clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=case["kl"],
                               scale=s["scale"], grad_dtype=grad)
        return {"loss": r.loss, "row_loss": r.row_loss, "logp": r.logp, "dlogits": r.dlogits}
    if op == "preference":
        r = losses.preference_loss(s["z"], s["tokens"], s["seq_off"], ref_logp=s["ref_logp"],
                                   weight=s["weight"], temperature=tau, beta=BETA,
                                   label_smoothing=SMOOTHING, scale=s["scale"], grad_dtype=grad)
        return {"loss": r.loss, "pair_loss": r.pair_loss, "margin": r.margin, "logp": r.logp,
                "dlogits": r.dlogits}
    r = losses.distill_loss(s["z"], s["top_index"], s["top_logit"], teacher_lse=s["teacher_lse"],
                            weight=s["weight"], temperature=tau, scale=s["scale"], grad_dtype=grad)
    return {"loss": r.loss, "row_loss": r.row_loss, "dlogits": r.dlogits}


# ----------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    """From the definitions in 64 bits, 256 rows at a time."""
    s = prepare(case, seed)
    tau, w = case["tau"], s["weight"].double()
    T, parts = case["rows"], []
    coef = None
    if case["op"] == "preference":
        first = _exact_logp(s, 0, T)
        live, pair = [], []
        coef = torch.zeros(T, dtype=torch.float64, device=w.device)
        dif = w * (first - s["ref_logp"].double())
        for i in range(case["pairs"]):
            a, b, c = s["seq_off"][2 * i:2 * i + 3]
            m = BETA * (dif[a:b].sum() - dif[b:c].sum())
            sig = torch.sigmoid(m)
            pair.append(-(1 - SMOOTHING) * torch.nn.functional.logsigmoid(m)
                        - SMOOTHING * torch.nn.functional.logsigmoid(-m))
            live.append(m)
            dm = BETA * s["scale"] * (sig - (1 - SMOOTHING))
            coef[a:b] = dm * w[a:b]
            coef[b:c] = -dm * w[b:c]
        used = (w != 0) & (torch.arange(T, device=w.device) < s["seq_off"][-1])
        out = {"pair_loss": torch.stack(pair), "margin": torch.stack(live),
               "loss": s["scale"] * torch.stack(pair).sum(), "logp": first * used}
    for a in range(0, T, 256):
        b = min(T, a + 256)
        parts.append(EXACT[case["op"]](s, a, b, coef))
    joined = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    if case["op"] == "preference":
        return {**out, **joined}
    if case["op"] in ("policy", "distill"):
        joined["loss"] = s["scale"] * joined["row_loss"].sum()
    return joined


def _exact_x(s, a, b):
    x = s["z"][a:b].double() / s["case"]["tau"]
    return x, torch.logsumexp(x, 1)


def _exact_logp(s, a, b):
    out = []
    for i in range(a, b, 256):
        x, lse = _exact_x(s, i, min(b, i + 256))
        out.append(x.gather(1, s["tokens"][i:i + 256, None])[:, 0] - lse)
    return torch.cat(out)


def _exact_dz(x, lse, tokens, dlogp, tau):
    hot = torch.zeros_like(x)
    hot.scatter_(1, tokens[:, None], 1.0)
    return (dlogp / tau)[:, None] * (hot - torch.softmax(x, 1))


def _exact_of_logp(s, a, b, coef):
    x, lse = _exact_x(s, a, b)
    live = s["weight"][a:b] != 0
    return {"logp": (x.gather(1, s["tokens"][a:b, None])[:, 0] - lse) * live, "lse": lse * live}


def _exact_of_logp_backward(s, a, b, coef):
    x, lse = _exact_x(s, a, b)
    return {"dlogits": _exact_dz(x, lse, s["tokens"][a:b], s["dlogp"][a:b].double(),
                                 s["case"]["tau"])}


def _exact_of_policy(s, a, b, coef):
    case, tau = s["case"], s["case"]["tau"]
    x, lse = _exact_x(s, a, b)
    tok, w = s["tokens"][a:b], s["weight"][a:b].double()
    lp = (x.gather(1, tok[:, None])[:, 0] - lse).requires_grad_()
    adv = s["advantage"][a:b].double()
    ratio = torch.exp(lp - s["old_logp"][a:b].double())
    l = -torch.min(ratio * adv, torch.clamp(ratio, 1 - CLIP_LOW, 1 + CLIP_HIGH) * adv)
    if s["ref_logp"] is not None:
        gap = s["ref_logp"][a:b].double() - lp
        l = l + case["kl"] * (torch.exp(gap) - gap - 1)
    (d,) = torch.autograd.grad((w * l).sum(), lp)
    return {"row_loss": (w * l).detach(), "logp": lp.detach() * (w != 0),
            "dlogits": _exact_dz(x, lse, tok, s["scale"] * d, tau)}


def _exact_of_preference(s, a, b, coef):
    x, lse = _exact_x(s, a, b)
    return {"dlogits": _exact_dz(x, lse, s["tokens"][a:b], coef[a:b], s["case"]["tau"])}


def _exact_of_distill(s, a, b, coef):
    case, tau, w = s["case"], s["case"]["tau"], s["weight"][a:b].double()
    z = s["z"][a:b].double().requires_grad_()
    index = s["top_index"][a:b].long()
    lp = torch.log_softmax(z / tau, 1)
    y = s["top_logit"][a:b].double() / tau
    if s["teacher_lse"] is None:
        lq = torch.log_softmax(y, 1)
        l = (lq.exp() * (lq - lp.gather(1, index))).sum(1)
    else:
        lq = y - s["teacher_lse"][a:b].double()[:, None]
        q = lq.exp()
        qr = (1 - q.sum(1)).clamp(min=0)
        out = torch.zeros_like(z, dtype=torch.bool).scatter_(1, index, True)
        lr = torch.logsumexp(lp.masked_fill(out, -math.inf), 1)
        l = (q * (lq - lp.gather(1, index))).sum(1) + torch.xlogy(qr, qr) - qr * lr
    l = w * tau * tau * l
    (d,) = torch.autograd.grad(s["scale"] * l.sum(), z)
    return {"row_loss": l.detach(), "dlogits": d}


EXACT = {"logp": _exact_of_logp, "logp_backward": _exact_of_logp_backward,
         "policy": _exact_of_policy, "preference": _exact_of_preference,
         "distill": _exact_of_distill}
