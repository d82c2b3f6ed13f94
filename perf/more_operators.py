"""Measured work of the two ends of a model around the feed-forward blocks: the
token embedding in front of them and the vocabulary loss behind them.

  kind            one pass
  embed_fwd       y = scale * weight[ids]: serving, or the forward half of a step
  embed_train     forward and backward: y, d_weight (the tokens of one id summed)
  xent_eval       softmax cross entropy of hidden @ weight^T, a value per token (scoring)
  xent_train      forward and backward: loss, d_hidden, d_weight; logits are not kept
  distill_eval    divergence from a teacher's top logits, a value per token
  distill_train   forward and backward of it: loss, d_hidden, d_weight

Sizes are this repository's blocks (fusionllm_amd/configs.py: dim 768 and 2048,
up to 32768 tokens) and generic vocabularies and odd sizes around them.  With
``own`` false ``run`` computes the plain form in fp32 (losses summed in fp64);
with ``own`` true it calls the framework.
"""
import math

import torch

own = False

IGNORE = -100
W_STD = 0.02
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one token of one user: a serving step, latency only
        {"name": "embed_fwd_t1_d768", "kind": "embed_fwd", "tokens": 1, "dim": 768, "vocab": 32768, "dtype": "bf16",
         "scale": 1.0, "pad": 0.0},
        # a ragged prompt, rows scaled by sqrt(dim) on their way into the residual stream
        {"name": "embed_fwd_t601_d2048", "kind": "embed_fwd", "tokens": 601, "dim": 2048, "vocab": 50021,
         "dtype": "bf16", "scale": 45.25, "pad": 0.0},
        # the headline training batch, 8 x 2048 tokens of dim 768, a fifth of them padding; odd vocabulary
        {"name": "embed_train_t16384_d768", "kind": "embed_train", "tokens": 16384, "dim": 768, "vocab": 50021,
         "dtype": "bf16", "scale": 27.75, "pad": 0.2},
        # the many-expert block's batch in the trainer's setting: fp32 parameters, a large vocabulary
        {"name": "embed_train_t32768_d2048", "kind": "embed_train", "tokens": 32768, "dim": 2048, "vocab": 131072,
         "dtype": "fp32", "scale": 1.0, "pad": 0.0},
        # scoring the few answer tokens of one prompt: latency and one read of the weight
        {"name": "xent_eval_t37_d768", "kind": "xent_eval", "tokens": 37, "dim": 768, "vocab": 32768, "dtype": "bf16",
         "drop": 0.0, "reduction": "none", "logit_scale": 1.0},
        # the headline training batch before an odd vocabulary
        {"name": "xent_train_t16384_d768", "kind": "xent_train", "tokens": 16384, "dim": 768, "vocab": 50021,
         "dtype": "bf16", "drop": 0.0, "reduction": "mean", "logit_scale": 1.0},
        # fine-tuning: prompt tokens carry no loss; odd in every direction
        {"name": "xent_train_t4099_d1001", "kind": "xent_train", "tokens": 4099, "dim": 1001, "vocab": 32003,
         "dtype": "bf16", "drop": 0.4, "reduction": "sum", "logit_scale": 0.75},
        # the many-expert block's batch before a large vocabulary
        {"name": "xent_train_t32768_d2048", "kind": "xent_train", "tokens": 32768, "dim": 2048, "vocab": 131072,
         "dtype": "bf16", "drop": 0.0, "reduction": "mean", "logit_scale": 1.0},
        # fp32 operands, kept in fp32 precision throughout
        {"name": "xent_train_fp32_t2047_d768", "kind": "xent_train", "tokens": 2047, "dim": 768, "vocab": 32768,
         "dtype": "fp32", "drop": 0.1, "reduction": "mean", "logit_scale": 1.0},
        # a micro-batch of distillation from a teacher's 64 largest logits
        {"name": "distill_train_t4096_d2048", "kind": "distill_train", "tokens": 4096, "dim": 2048, "vocab": 65536,
         "dtype": "bf16", "drop": 0.0, "reduction": "mean", "logit_scale": 1.0, "top": 64, "temperature": 2.0},
        # lists of different lengths (a teacher cut by probability), token weights applied behind
        {"name": "distill_train_t1021_d768", "kind": "distill_train", "tokens": 1021, "dim": 768, "vocab": 50021,
         "dtype": "bf16", "drop": 0.25, "reduction": "none", "logit_scale": 1.0, "top": 100, "temperature": 1.0},
        # the divergence of one sequence, validation
        {"name": "distill_eval_t300_d768", "kind": "distill_eval", "tokens": 300, "dim": 768, "vocab": 32768,
         "dtype": "bf16", "drop": 0.1, "reduction": "none", "logit_scale": 1.0, "top": 32, "temperature": 1.0},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["embed_fwd", "embed_train", "xent_eval", "xent_train", "xent_train", "distill_eval",
                       "distill_train"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    dim = _log_int(rng, 48, 4096)
    if rng.random() < 0.6:
        dim = -(-dim // 64) * 64
    vocab = _log_int(rng, 1000, 131072)
    if rng.random() < 0.5:
        vocab = min(131072, -(-vocab // 64) * 64)
    if kind.startswith("embed"):
        most = min(65536, (32768 * 2048) // dim)
        if vocab * dim > 131072 * 2048:
            vocab = 131072 * 2048 // dim
        return {"kind": kind, "tokens": _log_int(rng, 1, most), "dim": dim, "vocab": vocab, "dtype": dtype,
                "scale": rng.choice([1.0, 1.0, round(math.sqrt(dim), 2)]),
                "pad": rng.choice([0.0, 0.3]) if kind == "embed_train" else 0.0}
    budget = 32768 * 131072 * 2048 // 4
    if dtype == "fp32":
        budget //= 16
    most = max(1, min(32768, budget // (vocab * dim)))
    case = {"kind": kind, "tokens": _log_int(rng, 1, most), "dim": dim, "vocab": vocab, "dtype": dtype,
            "drop": rng.choice([0.0, 0.0, 0.15, 0.6]),
            "reduction": "none" if kind.endswith("eval") else rng.choice(["mean", "mean", "sum", "none"]),
            "logit_scale": rng.choice([1.0, 1.0, 0.5])}
    if kind.startswith("distill"):
        case["top"] = _log_int(rng, 1, 256)
        case["tokens"] = min(case["tokens"], 8192)
        case["temperature"] = rng.choice([1.0, 2.0, 3.5])
    return case


def _zipf(gen, n, vocab):
    """Token ids as text has them: frequency falls with the rank."""
    u = torch.rand(n, device="cuda", generator=gen, dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp_(0, vocab - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, T, D, V = DTYPES[case["dtype"]], case["tokens"], case["dim"], case["vocab"]
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)
    rand = lambda *shape: torch.rand(*shape, device="cuda", generator=gen)
    state = {"case": dict(case)}
    ids = _zipf(gen, T, V)
    weight = (W_STD * randn(V, D)).to(dtype)
    train = case["kind"].endswith("train")
    if case["kind"].startswith("embed"):
        state["pad"] = None
        if case["pad"] > 0:
            state["pad"] = V - 1
            ids[rand(T) < case["pad"]] = V - 1
        state["ids"] = ids
        if train:
            state["dy"] = (0.01 * randn(T, D)).to(dtype)
    else:
        # hidden states of a model that has learnt something: part noise, part the target's own row
        pull = rand(T, 1) * (12.0 / (D * W_STD * W_STD))
        hidden = randn(T, D) * (0.5 + rand(T, 1)) + pull * weight[ids].float()
        state["hidden"] = hidden.to(dtype).requires_grad_(train)
        lost = torch.randperm(T, device="cuda", generator=gen)[:int(T * case["drop"])]
        if case["kind"].startswith("xent"):
            ids[lost] = IGNORE
            state["target"] = ids
        else:
            K = min(case["top"], V)
            steps = torch.randint(1, max(2, V // K), (T, K), device="cuda", generator=gen)
            index = (ids[:, None] + steps.cumsum(1) - steps) % V  # distinct; the first is the target
            # falling logits, as a sorted list of the largest is
            logits = 14.0 - 1.5 * (-torch.log1p(-0.98 * rand(T, K))).cumsum(1)
            if case["drop"] > 0:  # lists of different lengths, some empty
                length = torch.randint(1, K + 1, (T, 1), device="cuda", generator=gen)
                length[lost] = 0
                index = torch.where(torch.arange(K, device="cuda") < length, index, IGNORE)
            state["index"], state["teacher"] = index, logits
        if train and case["reduction"] == "none":
            state["dloss"] = rand(T) / T
    state["weight"] = weight.requires_grad_(train)
    return state


# ---- plain forms --------------------------------------------------------------


def _plain_embed(state):
    case, w, ids = state["case"], state["weight"].detach(), state["ids"]
    out = {"y": (w[ids].float() * case["scale"]).to(w.dtype)}
    if case["kind"] == "embed_train":
        dy = state["dy"].float() * case["scale"]
        if state["pad"] is not None:
            dy = torch.where((ids == state["pad"])[:, None], 0.0, dy)
        dw = torch.zeros(w.shape, dtype=torch.float32, device="cuda")
        out["d_weight"] = dw.index_add_(0, ids, dy).to(w.dtype)
    return out


def _plain_loss(state):
    """Pieces of the tokens against the whole vocabulary: logits, softmax, gradients."""
    case = state["case"]
    h, w = state["hidden"].detach(), state["weight"].detach()
    T, V = h.shape[0], w.shape[0]
    train, distill = case["kind"].endswith("train"), case["kind"].startswith("distill")
    tau = case["temperature"] if distill else 1.0
    factor = case["logit_scale"] / tau
    wf = w.float()
    wt = wf.t().contiguous()
    if distill:
        index = state["index"]
        there = index != IGNORE
        teacher = torch.where(there, state["teacher"].float() / tau, -math.inf)
        rows = there.any(1)
        peak = torch.where(rows, teacher.amax(1), 0.0)
        q = torch.exp(teacher - peak[:, None])
        q = q / torch.where(rows, q.sum(1), 1.0)[:, None]
        log_q = torch.where(q > 0, torch.log(torch.where(q > 0, q, 1.0)), 0.0)
    else:
        index = state["target"][:, None]
        rows = index[:, 0] != IGNORE
        q, log_q = rows[:, None].float(), 0.0
    index = index.clamp_min(0)
    count = rows.sum()
    if case["reduction"] == "none":
        up = state["dloss"] if train else None
    elif case["reduction"] == "mean":
        up = (1.0 / count).float().expand(T)
    else:
        up = torch.ones(T, device="cuda")
    loss = torch.empty(T, device="cuda")
    dh, dw = (torch.empty(h.shape, device="cuda"), torch.zeros(w.shape, device="cuda")) if train else (None, None)
    piece = max(1, min(T, (1 << 29) // V))
    for a in range(0, T, piece):
        b = min(T, a + piece)
        hf = h[a:b].float()
        s = (hf @ wt).mul_(factor)
        s = s - s.amax(1, keepdim=True)
        e = torch.exp(s)
        total = e.sum(1, keepdim=True)
        log_p = s.gather(1, index[a:b]) - torch.log(total)
        lq = log_q[a:b] if distill else 0.0
        loss[a:b] = (q[a:b] * (lq - log_p)).sum(1) * (tau * tau)
        if train:
            g = e.div_(total) * rows[a:b, None]
            g.scatter_add_(1, index[a:b], -q[a:b])
            g.mul_((up[a:b] * (tau * tau * factor))[:, None])
            dh[a:b] = g @ wf
            dw += g.t() @ hf
    loss = torch.where(rows, loss, 0.0)
    if case["reduction"] == "mean":
        loss = (loss.double().sum() / count).float()
    elif case["reduction"] == "sum":
        loss = loss.double().sum().float()
    out = {"loss": loss}
    if train:
        out["d_hidden"], out["d_weight"] = dh.to(h.dtype), dw.to(w.dtype)
    return out


# ---- the framework's operators ------------------------------------------------


def _own_embed(state):
    import fusionllm_amd
    case, w = state["case"], state["weight"]
    y = fusionllm_amd.embedding(state["ids"], w, scale=case["scale"], padding_idx=state["pad"])
    if case["kind"] == "embed_fwd":
        return {"y": y}
    dw, = torch.autograd.grad(y, [w], state["dy"])
    return {"y": y.detach(), "d_weight": dw}


def _own_loss(state):
    import fusionllm_amd
    case, h, w = state["case"], state["hidden"], state["weight"]
    options = dict(ignore_index=IGNORE, reduction=case["reduction"], logit_scale=case["logit_scale"])
    if case["kind"].startswith("xent"):
        loss = fusionllm_amd.linear_cross_entropy(h, w, state["target"], **options)
    else:
        loss = fusionllm_amd.linear_distillation(h, w, state["index"], state["teacher"],
                                                 temperature=case["temperature"], **options)
    if not case["kind"].endswith("train"):
        return {"loss": loss}
    dh, dw = torch.autograd.grad(loss, [h, w], state.get("dloss"))
    return {"loss": loss.detach(), "d_hidden": dh, "d_weight": dw}


def run(state):
    if state["case"]["kind"].startswith("embed"):
        return _own_embed(state) if own else _plain_embed(state)
    return _own_loss(state) if own else _plain_loss(state)


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    T, D, V = case["tokens"], case["dim"], case["vocab"]
    train = case["kind"].endswith("train")
    if case["kind"].startswith("embed"):
        # a row read and a row written per token; the output's gradient in, the weight's whole gradient out
        return {"bytes": T * (8 + 2 * D * size) + (T * D * size + V * D * size if train else 0),
                "flops": T * D * (2 if train else 1)}
    rows = T - int(T * case["drop"])
    lists = T * (12 * min(case["top"], V) if case["kind"].startswith("distill") else 8)
    # the logits; their product with the weight, and with the hidden states, for the gradients
    flops = (6 if train else 2) * rows * D * V
    return {"bytes": (2 if train else 1) * (T + V) * D * size + lists + 4 * T, "flops": flops}


# ---- the operators' definitions in 64 bits ------------------------------------


def _exact_embed(case, state):
    w, ids = state["weight"].detach().double(), state["ids"]
    out = {"y": torch.nn.functional.one_hot(ids, w.shape[0]).double() @ w * case["scale"] if len(ids) < 8
           else torch.index_select(w, 0, ids).mul_(case["scale"])}
    if case["kind"] == "embed_train":
        # tokens of one id lie together after a sort: differences of running sums are too coarse, so
        # each id's rows are reduced as a segment
        keep = ids != (-1 if state["pad"] is None else state["pad"])
        order = torch.argsort(ids[keep], stable=True)
        dy = state["dy"].double()[keep][order]
        lengths = torch.bincount(ids[keep], minlength=w.shape[0])
        out["d_weight"] = torch.segment_reduce(dy, "sum", lengths=lengths, axis=0, initial=0.0) * case["scale"]
    return out


def _exact_loss(case, state):
    """Softmax by logaddexp over the valid tokens alone, gradients as matrices of probabilities less targets."""
    h, w = state["hidden"].detach().double(), state["weight"].detach().double()
    train, distill = case["kind"].endswith("train"), case["kind"].startswith("distill")
    T, V = h.shape[0], w.shape[0]
    tau = case["temperature"] if distill else 1.0
    lists = state["index"] if distill else state["target"].view(-1, 1)
    valid = torch.nonzero((lists >= 0).any(1)).view(-1)
    n = len(valid)
    share = {"none": state["dloss"].double() if "dloss" in state else None,
             "mean": torch.full((T,), 1.0 / max(n, 1), device="cuda", dtype=torch.float64),
             "sum": torch.ones(T, device="cuda", dtype=torch.float64)}[case["reduction"]]
    losses = torch.zeros(T, device="cuda", dtype=torch.float64)
    dh, dw = torch.zeros_like(h) if train else None, torch.zeros_like(w) if train else None
    for part in valid.split(max(1, (1 << 27) // V)):
        x = h[part]
        z = torch.matmul(x, w.T) * (case["logit_scale"] / tau)
        log_p = z - torch.logsumexp(z, 1, keepdim=True)
        picked = lists[part]
        if distill:
            t = state["teacher"][part].double() / tau
            t = t.masked_fill(picked < 0, -math.inf)
            log_t = t - torch.logsumexp(t, 1, keepdim=True)
            prob = log_t.exp()
            at = log_p.gather(1, picked.clamp(min=0))
            losses[part] = tau ** 2 * torch.where(picked < 0, 0.0, prob * (log_t - at)).nan_to_num(0.0).sum(1)
        else:
            prob = torch.ones_like(picked, dtype=torch.float64)
            losses[part] = -log_p.gather(1, picked)[:, 0]
        if train:
            delta = log_p.exp_()
            row, col = torch.nonzero(picked >= 0, as_tuple=True)
            delta.index_put_((row, picked[row, col]), -prob[row, col], accumulate=True)
            delta *= (share[part] * tau * case["logit_scale"])[:, None]
            dh[part] = torch.matmul(delta, w)
            dw += torch.matmul(delta.T, x)
    total = {"none": losses, "sum": losses.sum(), "mean": losses.sum() / n if n else losses.sum() * math.nan}
    out = {"loss": total[case["reduction"]]}
    if train:
        out["d_hidden"], out["d_weight"] = dh, dw
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return (_exact_embed if case["kind"].startswith("embed") else _exact_loss)(case, state)
