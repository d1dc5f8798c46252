"""Cases that measure the closed-loop fine-tuning operators (prosim_amd.finetune): the log-probability of a drawn choice, the clipped policy loss
with its KL term, the pairwise preference loss and the clipping of a gradient list by its global norm.

``own`` = False computes the plain form with elementary torch operations, ``own`` = True calls the framework.  Rows are decisions (replan x agent, or
token positions), the last axis is what is chosen from: motion modes, or a vocabulary of motion tokens.
"""
import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
MAX_ELEMENTS = 1 << 28          # the largest listed logits and gradient list


def listed():
    return [
        # ---- choice_logp
        # 8 replans x 128 agents of one scene choosing among 3 motion modes: what a rollout records, and its gradient (latency)
        {"name": "logp_modes", "op": "choice_logp", "rows": 1024, "choices": 3, "dtype": "float32", "train": True, "valid": 1.0},
        # a single decision over a large vocabulary while serving: one long row
        {"name": "logp_single", "op": "choice_logp", "rows": 1, "choices": 131072, "dtype": "bfloat16", "train": False, "valid": 1.0},
        # the reference policy's log-probabilities over an odd vocabulary, padded rows among them (forward only)
        {"name": "logp_reference", "op": "choice_logp", "rows": 3001, "choices": 50021, "dtype": "float16", "train": False, "valid": 0.9},
        # a training batch of token positions, forward and backward
        {"name": "logp_train", "op": "choice_logp", "rows": 8192, "choices": 32768, "dtype": "bfloat16", "train": True, "valid": 0.95},
        # ---- policy_loss
        # 8 replans x 8 scenes x 128 agents choosing among 64 goals (the most the goal head offers), entering / leaving agents masked
        {"name": "policy_goals", "op": "policy_loss", "rows": 8192, "choices": 64, "dtype": "float32", "valid": 0.9, "kl_coef": 0.05},
        # a vocabulary of 2048 motion tokens plus one for "parked"; single precision
        {"name": "policy_tokens", "op": "policy_loss", "rows": 5119, "choices": 2049, "dtype": "float32", "valid": 1.0, "kl_coef": 0.0},
        # few long rows: the last micro-batch of an epoch
        {"name": "policy_few", "op": "policy_loss", "rows": 7, "choices": 100003, "dtype": "float16", "valid": 1.0, "kl_coef": 0.02},
        # the largest: long rows, masked padding, KL to a reference policy
        {"name": "policy_vocab", "op": "policy_loss", "rows": 2048, "choices": 131072, "dtype": "bfloat16", "valid": 0.9, "kl_coef": 0.04},
        # ---- preference_loss
        # 16 pairs of rollouts (better / worse replica of an agent), 8 replans each
        {"name": "pairs_replans", "op": "preference_loss", "pairs": 16, "steps": 8, "valid": 1.0},
        # long ragged token sequences
        {"name": "pairs_long", "op": "preference_loss", "pairs": 1024, "steps": 4093, "valid": 0.7},
        # ---- clip_grads
        # the parameter list of the demo model: 1226 tensors, 11.4 M elements
        {"name": "clip_demo", "op": "clip_grads", "tensors": 1226, "elements": 11399220, "dtype": "float32", "max_norm": 1.0},
        # a large model's gradients in half the bytes
        {"name": "clip_large", "op": "clip_grads", "tensors": 292, "elements": MAX_ELEMENTS, "dtype": "bfloat16", "max_norm": 1.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["choice_logp", "policy_loss", "policy_loss", "preference_loss", "clip_grads"])
    if op == "preference_loss":
        steps = _log_int(rng, 1, 4096)
        return {"op": op, "pairs": _log_int(rng, 1, max(1, min(4096, 1024 * 4093 // steps))), "steps": steps, "valid": rng.choice([1.0, 0.7])}
    if op == "clip_grads":
        n = _log_int(rng, 1, 1300)
        return {"op": op, "tensors": n, "elements": _log_int(rng, max(n, 1000), MAX_ELEMENTS), "dtype": rng.choice(sorted(DTYPES)),
                "max_norm": rng.choice([0.5, 1.0, 1.0e5])}
    k = _log_int(rng, 2, 131072)
    dtype = rng.choice(sorted(DTYPES))
    cap = MAX_ELEMENTS // (2 if dtype == "float32" else 1)      # the bytes of the largest listed case
    case = {"op": op, "rows": _log_int(rng, 1, max(1, min(65536, cap // k))), "choices": k, "dtype": dtype, "valid": rng.choice([1.0, 0.9])}
    if op == "choice_logp":
        case["train"] = rng.random() < 0.6
    else:
        case["kl_coef"] = rng.choice([0.0, 0.04])
    return case


def _tensor_sizes(n, total):
    """Ragged sizes over several orders of magnitude, at least one element each, ``total`` in all."""
    rng = random.Random(n * 1000003 + total)
    share = [math.exp(rng.uniform(0.0, 7.0)) for _ in range(n)]
    scale = (total - n) / sum(share)
    sizes = [1 + int(s * scale) for s in share]
    sizes[-1] += total - sum(sizes)
    return sizes


def _decisions(case, gen, dev):
    rows, k = case["rows"], case["choices"]
    logits = torch.empty((rows, k), dtype=DTYPES[case["dtype"]], device=dev)
    step = max(1, (1 << 26) // k)
    for a in range(0, rows, step):
        b = min(rows, a + step)
        logits[a:b] = torch.randn((b - a, k), generator=gen, device=dev) * 2.0
    choice = torch.randint(0, k, (rows,), generator=gen, device=dev)
    # a drawn choice is a likely one: between e^-4 and 1 or so
    bump = math.log(k) + 2.0 + 1.5 * torch.randn((rows,), generator=gen, device=dev)
    logits.scatter_(1, choice[:, None], bump[:, None].to(logits.dtype))
    mask = None
    if case["valid"] < 1.0:
        mask = torch.rand((rows,), generator=gen, device=dev) < case["valid"]
        choice = torch.where(mask, choice, torch.zeros_like(choice))
    return logits, choice, mask


def _recorded_logp(logits, choice):
    out = torch.empty(logits.shape[0], device=logits.device)
    step = max(1, (1 << 26) // logits.shape[1])
    for a in range(0, logits.shape[0], step):
        x = logits[a:a + step].float()
        out[a:a + step] = x.gather(1, choice[a:a + step, None])[:, 0] - torch.logsumexp(x, 1)
    return out


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    op = case["op"]
    st = {"case": case}
    if op in ("choice_logp", "policy_loss"):
        logits, choice, mask = _decisions(case, gen, dev)
        rows = case["rows"]
        if op == "choice_logp":
            st["grad_out"] = torch.randn((rows,), generator=gen, device=dev) / rows
        else:
            now = _recorded_logp(logits, choice)
            # the policy moved a little since the rollout, and more since the reference policy
            st["old_logp"] = now + 0.15 * torch.randn((rows,), generator=gen, device=dev)
            st["ref_logp"] = now + 0.4 * torch.randn((rows,), generator=gen, device=dev) if case["kl_coef"] > 0 else None
            st["advantage"] = torch.randn((rows,), generator=gen, device=dev)
        st["choice"], st["mask"] = choice, mask
        st["logits"] = logits.requires_grad_(op == "policy_loss" or case["train"])
    elif op == "preference_loss":
        shape = (case["pairs"], case["steps"])
        for side, shift in (("better", 0.05), ("worse", -0.05)):
            ref = -2.0 * torch.rand(shape, generator=gen, device=dev)
            st[side + "_ref"] = ref
            st[side] = (ref + shift / math.sqrt(shape[1]) + 0.3 * torch.randn(shape, generator=gen, device=dev)).requires_grad_(True)
            length = None
            if case["valid"] < 1.0:     # sequences end at lengths of their own
                length = (torch.rand((shape[0], 1), generator=gen, device=dev) * 2.0 * case["valid"] * shape[1]).long().clamp(max=shape[1])
                length = torch.arange(shape[1], device=dev)[None, :] < length
            st[side + "_mask"] = length
    else:
        flat = torch.empty(case["elements"], dtype=DTYPES[case["dtype"]], device=dev)
        for a in range(0, flat.numel(), 1 << 26):
            part = flat[a:a + (1 << 26)]
            part.copy_(torch.randn(part.shape, generator=gen, device=dev) * 0.01)
        # data-parallel training keeps gradients as views of one flat buffer, whatever alignment that gives; a short list has tensors of their own
        st["grads"] = list(flat.split(_tensor_sizes(case["tensors"], case["elements"])))
        st["held"] = [flat]
        if case["tensors"] <= 32:
            st["grads"] = st["held"] = [g.clone() for g in st["grads"]]
    return st


# ---- the plain forms -----------------------------------------------------------------------------------------------

def _plain_row_stats(x, choice):
    m = x.max(1, keepdim=True).values
    e = torch.exp(x - m)
    s = e.sum(1, keepdim=True, dtype=torch.float64)      # 64 bits: the ratio is compared with the borders of the clipping range
    logp = (x.gather(1, choice[:, None]) - m).double() - torch.log(s)
    return e, s, logp[:, 0]


def _plain_row_grad(e, s, choice, coef, dtype):
    g = e / s.float() * (-coef[:, None])
    g.scatter_add_(1, choice[:, None], coef[:, None])
    return g.to(dtype)


def _plain_choice_logp(st):
    logits, choice, mask = st["logits"].detach(), st["choice"], st["mask"]
    e, s, logp = _plain_row_stats(logits.float(), choice)
    if mask is not None:
        logp = torch.where(mask, logp, torch.zeros_like(logp))
    out = [logp.float()]
    if st["case"]["train"]:
        coef = st["grad_out"] if mask is None else torch.where(mask, st["grad_out"], torch.zeros_like(st["grad_out"]))
        out.append(_plain_row_grad(e, s, choice, coef, logits.dtype))
    return out


def _plain_policy_loss(st):
    logits, choice, mask, beta = st["logits"].detach(), st["choice"], st["mask"], st["case"]["kl_coef"]
    e, s, logp = _plain_row_stats(logits.float(), choice)
    valid = torch.ones_like(choice, dtype=torch.bool) if mask is None else mask
    n = valid.sum().clamp(min=1).double()
    adv = st["advantage"].double()
    r = torch.exp(logp - st["old_logp"].double())
    s1, s2 = r * adv, r.clamp(1.0 - 0.2, 1.0 + 0.28) * adv
    clipped = s2 < s1
    loss, d_logp = -torch.where(clipped, s2, s1), torch.where(clipped, torch.zeros_like(r), -s1)
    kl = torch.zeros_like(r)
    if st["ref_logp"] is not None:
        d = st["ref_logp"].double() - logp
        kl = torch.exp(d) - d - 1.0
        loss, d_logp = loss + beta * kl, d_logp + beta * (1.0 - torch.exp(d))
    zero = torch.zeros_like(r)
    loss, kl, d_logp, logp = (torch.where(valid, v, zero) for v in (loss, kl, d_logp, logp))
    frac = (clipped & valid).sum().double() / n
    grad = _plain_row_grad(e, s, choice, (d_logp / n).float(), logits.dtype)
    return [(loss.sum() / n).float(), logp.float(), (kl.sum() / n).float(), frac.float(), grad]


def _plain_preference_loss(st):
    zero = torch.zeros((), dtype=torch.float64, device=st["better"].device)
    h, masks = 0.0, []
    for side, sign in (("better", 1.0), ("worse", -1.0)):
        d = st[side].detach().double() - st[side + "_ref"].double()      # 64 bits: sums of thousands of terms
        if st[side + "_mask"] is not None:
            d = torch.where(st[side + "_mask"], d, zero)
        h = h + sign * d.sum(1)
        masks.append(st[side + "_mask"])
    beta, eps, pairs = 0.1, 0.05, st["case"]["pairs"]
    z = beta * h
    up, down = 1.0 / (1.0 + torch.exp(-z)), 1.0 / (1.0 + torch.exp(z))
    soft = torch.clamp(z, min=0.0) + torch.log1p(torch.exp(-z.abs()))    # -ln sigmoid(-z)
    loss = ((1.0 - eps) * (soft - z) + eps * soft).sum() / pairs
    coef = (-beta * ((1.0 - eps) * down - eps * up) / pairs)[:, None]
    grads = []
    for mask, sign in zip(masks, (1.0, -1.0)):
        g = (sign * coef).expand(pairs, st["case"]["steps"])
        grads.append((g.clone() if mask is None else torch.where(mask, g, zero)).float())
    return [loss.float(), z.float()] + grads


def _plain_clip_grads(st):
    total = sum(torch.sum(g.float() * g.float()) for g in st["grads"])
    norm = torch.sqrt(total)
    coef = torch.clamp(st["case"]["max_norm"] / (norm + 1.0e-6), max=1.0)
    for g in st["grads"]:
        g.copy_(g.float() * coef)
    return [norm] + st["held"]


# ---- one pass ------------------------------------------------------------------------------------------------------

def run(st):
    case = st["case"]
    op = case["op"]
    if not own:
        with torch.no_grad():
            return {"choice_logp": _plain_choice_logp, "policy_loss": _plain_policy_loss, "preference_loss": _plain_preference_loss,
                    "clip_grads": _plain_clip_grads}[op](st)
    from prosim_amd import finetune
    if op == "choice_logp":
        logp = finetune.choice_logp(st["logits"], st["choice"], mask=st["mask"])
        if not case["train"]:
            return [logp]
        grad, = torch.autograd.grad(logp, st["logits"], st["grad_out"])
        return [logp.detach(), grad]
    if op == "policy_loss":
        out = finetune.policy_loss(st["logits"], st["choice"], st["old_logp"], st["advantage"], ref_logp=st["ref_logp"], mask=st["mask"],
                                   clip_low=0.2, clip_high=0.28, kl_coef=case["kl_coef"])
        grad, = torch.autograd.grad(out.loss, st["logits"])
        return [out.loss.detach(), out.logp, out.kl, out.clip_frac, grad]
    if op == "preference_loss":
        out = finetune.preference_loss(st["better"], st["worse"], st["better_ref"], st["worse_ref"], better_mask=st["better_mask"],
                                       worse_mask=st["worse_mask"], beta=0.1, label_smoothing=0.05)
        grads = torch.autograd.grad(out.loss, (st["better"], st["worse"]))
        return [out.loss.detach(), out.margin, *grads]
    norm = finetune.clip_grads_(st["grads"], case["max_norm"])
    return [norm] + st["held"]


def work(case):
    """Each input read once, each output written once; logits of masked rows are nobody's input."""
    op = case["op"]
    if op == "preference_loss":
        n = case["pairs"] * case["steps"]
        masks = 2 if case["valid"] < 1.0 else 0
        return {"bytes": n * (4 * 4 + 2 * 4 + masks) + 8 * case["pairs"], "flops": 6 * n}
    if op == "clip_grads":
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": 2 * size * case["elements"], "flops": 3 * case["elements"]}
    size = 4 if case["dtype"] == "float32" else 2
    rows, n = case["rows"], case["rows"] * case["choices"]
    masked = 1 if case["valid"] < 1.0 else 0
    by = int(case["valid"] * n) * size + rows * (8 + 4 + masked)
    fl = 4 * int(case["valid"] * n)
    if op == "policy_loss":
        by += n * size + rows * (12 if case["kl_coef"] > 0 else 8)
        fl += 3 * n
    elif case["train"]:
        by += n * size + 4 * rows
        fl += 3 * n
    return {"bytes": by, "flops": fl}


# ---- the definition, in 64 bits -------------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "clip_grads":
            flat = [g.double() for g in st["held"]]
            norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g) for g in flat]))
            if float(norm) + 1.0e-6 <= case["max_norm"]:
                return [norm] + flat
            return [norm] + [g * (case["max_norm"] / (norm + 1.0e-6)) for g in flat]
        if op == "preference_loss":
            ratio = {}
            ones = torch.ones((case["pairs"], case["steps"]), dtype=torch.float64, device=st["better"].device)
            for side in ("better", "worse"):
                keep = ones if st[side + "_mask"] is None else st[side + "_mask"].double()
                ratio[side] = ((st[side].double() - st[side + "_ref"].double()) * keep).sum(1), keep
            z = 0.1 * (ratio["better"][0] - ratio["worse"][0])
            per = -0.95 * torch.nn.functional.logsigmoid(z) - 0.05 * torch.nn.functional.logsigmoid(-z)
            slope = 0.1 * (torch.sigmoid(z) - 0.95) / case["pairs"]          # d per / d h / P
            return [per.mean(), z, slope[:, None] * ratio["better"][1], -slope[:, None] * ratio["worse"][1]]
        rows, k = case["rows"], case["choices"]
        dev = st["choice"].device
        keep = torch.ones(rows, dtype=torch.float64, device=dev) if st["mask"] is None else st["mask"].double()
        idx = torch.arange(rows, device=dev)
        step = max(1, (1 << 25) // k)
        parts = range(0, rows, step)
        x = st["logits"].detach()
        logp = torch.cat([torch.log_softmax(x[a:a + step].double(), 1)[torch.arange(min(step, rows - a), device=dev), st["choice"][a:a + step]] for a in parts])
        if op == "choice_logp":
            outs, coef = [logp * keep], st["grad_out"].double() * keep
            if not case["train"]:
                return outs
        else:
            count = max(1.0, float(keep.sum()))
            ratio, adv = torch.exp(logp - st["old_logp"].double()), st["advantage"].double()
            free = ratio * adv
            held = torch.minimum(torch.maximum(ratio, torch.full_like(ratio, 0.8)), torch.full_like(ratio, 1.28)) * adv
            per, slope, kl = -torch.minimum(free, held), -free * (free <= held), torch.zeros_like(free)
            if st["ref_logp"] is not None:
                gap = logp - st["ref_logp"].double()
                kl = torch.expm1(-gap) + gap
                per, slope = per + case["kl_coef"] * kl, slope - case["kl_coef"] * torch.expm1(-gap)
            outs = [(per * keep).sum() / count, logp * keep, (kl * keep).sum() / count, ((held < free) * keep).sum() / count]
            coef = slope * keep / count
        grad = torch.empty((rows, k), dtype=torch.float64, device=dev)
        for a in parts:
            grad[a:a + step] = torch.softmax(x[a:a + step].double(), 1) * -coef[a:a + step, None]
        grad[idx, st["choice"]] += coef
        return outs + [grad]
