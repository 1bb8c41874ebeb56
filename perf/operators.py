"""The operators of token policies as they are measured: the teacher's top logits, the distillation loss with its gradient, the verification of drafts.

`run` computes them from elementary torch operations, or, where `own` is true, by the framework's entry points (cleanba_amd.tokens).  `exact` restates
each definition in 64 bits, apart from the plain forms."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
MOST_ELEMENTS = 3840 * 131072   # logits of the largest listed case


def listed():
    return [
        # the teacher answers one token: latency
        {"name": "top: one row", "op": "top", "rows": 1, "vocab": 131072, "k": 64, "dtype": "bf16", "temperature": 1.0, "masked": 0.0},
        # a rollout of 128 steps x 120 environments, 18 actions each: many tiny rows
        {"name": "top: rollout of 18 actions", "op": "top", "rows": 15360, "vocab": 18, "k": 4, "dtype": "f32", "temperature": 1.0, "masked": 0.1},
        # a minibatch of 3840 rows, a usual vocabulary
        {"name": "top: minibatch", "op": "top", "rows": 3840, "vocab": 32768, "k": 32, "dtype": "bf16", "temperature": 2.0, "masked": 0.0},
        # a vocabulary of odd size: rows start at any 2-byte address, a tenth of the tokens masked
        {"name": "top: odd vocabulary, masked", "op": "top", "rows": 1009, "vocab": 100003, "k": 128, "dtype": "f16", "temperature": 1.0, "masked": 0.1},
        # policy distillation (kickstarting) over 18 actions, one PPO minibatch
        {"name": "distill: 18 actions", "op": "distill", "rows": 3840, "vocab": 18, "k": 4, "dtype": "f32", "temperature": 1.0, "tail": True, "weights": True, "grad": True},
        # a few rows: latency of a training step's loss
        {"name": "distill: few rows", "op": "distill", "rows": 60, "vocab": 32768, "k": 32, "dtype": "bf16", "temperature": 1.0, "tail": False, "weights": False, "grad": True},
        # odd vocabulary in fp32, tail kept, a fifth of the rows is padding
        {"name": "distill: odd fp32, padded", "op": "distill", "rows": 777, "vocab": 50021, "k": 100, "dtype": "f32", "temperature": 2.0, "tail": True, "weights": True, "grad": True},
        # a whole minibatch over a large vocabulary
        {"name": "distill: minibatch", "op": "distill", "rows": 3840, "vocab": 131072, "k": 64, "dtype": "bf16", "temperature": 1.0, "tail": False, "weights": False, "grad": True},
        # one sequence being served
        {"name": "verify: one sequence", "op": "verify", "batch": 1, "drafts": 4, "vocab": 131072, "dtype": "bf16", "temperature": 1.0, "draft_logits": True, "ragged": False},
        # a serving batch, drafts of different lengths
        {"name": "verify: batch, ragged", "op": "verify", "batch": 64, "drafts": 8, "vocab": 131072, "dtype": "bf16", "temperature": 0.8, "draft_logits": True, "ragged": True},
        # 120 environments, seven drafted actions each
        {"name": "verify: 18 actions", "op": "verify", "batch": 120, "drafts": 7, "vocab": 18, "dtype": "f32", "temperature": 1.0, "draft_logits": True, "ragged": True},
        # drafts looked up rather than sampled (no draft distribution), odd vocabulary
        {"name": "verify: looked-up drafts, odd", "op": "verify", "batch": 37, "drafts": 5, "vocab": 50021, "dtype": "f16", "temperature": 1.0, "draft_logits": False, "ragged": True},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["top", "distill", "verify"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    vocab = _spread(rng, 2, 200000)
    if rng.random() < 0.3:
        vocab = max(8, vocab // 64 * 64)
    tau = rng.choice([0.7, 1.0, 1.0, 2.0])
    if op == "verify":
        drafts = rng.randint(0, 10)
        batch = _spread(rng, 1, max(1, min(512, MOST_ELEMENTS // 4 // ((2 * drafts + 1) * vocab))))
        return {"op": op, "batch": batch, "drafts": drafts, "vocab": vocab, "dtype": dtype, "temperature": tau, "draft_logits": rng.random() < 0.7, "ragged": rng.random() < 0.5}
    rows = _spread(rng, 1, max(1, min(16384, MOST_ELEMENTS // (2 if dtype == "f32" else 1) // vocab)))
    k = _spread(rng, 1, min(256, vocab))
    if op == "top":
        return {"op": op, "rows": rows, "vocab": vocab, "k": k, "dtype": dtype, "temperature": tau, "masked": rng.choice([0.0, 0.1])}
    return {"op": op, "rows": rows, "vocab": vocab, "k": k, "dtype": dtype, "temperature": tau, "tail": rng.random() < 0.5, "weights": rng.random() < 0.5, "grad": rng.random() < 0.75}


# ---------------------------------------------------------------------------------------- inputs
_ctx = None


def _context():
    """The context a program keeps: the smallest one the library makes."""
    global _ctx
    if _ctx is None:
        from cleanba_amd import lib
        cfg = lib.default_config(lib.ALGO_PPO)
        cfg.local_num_envs, cfg.num_actor_slots, cfg.num_steps, cfg.num_minibatches, cfg.update_epochs = 1, 1, 8, 1, 1
        _ctx = lib.Context(cfg)
    return _ctx


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _top_of(x, k):
    """Indices of the k largest of each row, equal ones by rising index: one whole number a logit, whose order is the order wanted."""
    vocab = x.shape[-1]
    bits = (x + 0.0).view(torch.int32)
    order = bits ^ ((bits >> 31) & 0x7FFFFFFF)
    key = (order.long() << 32) + torch.arange(vocab - 1, -1, -1, device=x.device)
    key = torch.topk(key, k, dim=-1).values
    return vocab - 1 - (key & 0xFFFFFFFF)


def prepare(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = dict(case)
    if own:
        state["ctx"] = _context()
    if case["op"] == "verify":
        # peaked logits (a few tokens hold most of the mass) of a target and of a draft that follows it
        batch, drafts, vocab = case["batch"], case["drafts"], case["vocab"]
        base = _normal(g, batch, drafts + 1, vocab) * 3.0
        state["target"] = (base + 0.4 * _normal(g, batch, drafts + 1, vocab)).to(dtype)
        state["draft"] = (base[:, :drafts] + 0.4 * _normal(g, batch, drafts, vocab)).to(dtype)
        # drafted tokens: sampled from the draft's distribution by exponential races
        race = torch.rand(batch, drafts, vocab, generator=g, device="cuda").clamp_(1e-12).log_().neg_().log_().neg_()
        state["tokens"] = (state["draft"].float() / case["temperature"] + race).argmax(-1).to(torch.int32) if drafts else torch.zeros(batch, 0, dtype=torch.int32, device="cuda")
        if not case["draft_logits"]:
            state["draft"] = None
        state["n_draft"] = torch.randint(0, drafts + 1, (batch,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None
        state["u_accept"] = torch.rand(batch, drafts, generator=g, device="cuda")
        state["u_sample"] = torch.rand(batch, generator=g, device="cuda")
        return state
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    teacher = _normal(g, rows, vocab) * 2.5
    if case["op"] == "top":
        if case["masked"]:
            teacher.masked_fill_(torch.rand(rows, vocab, generator=g, device="cuda") < case["masked"], -math.inf)
        state["logits"] = teacher.to(dtype)
        return state
    state["logits"] = (0.8 * teacher + _normal(g, rows, vocab)).to(dtype)
    step = max(1, (1 << 27) // vocab)
    state["teacher_idx"] = torch.cat([_top_of(teacher[i:i + step], k) for i in range(0, rows, step)]).to(torch.int32)
    state["teacher_logits"] = teacher.gather(1, state["teacher_idx"].long())
    state["teacher_lse"] = torch.logsumexp(teacher / case["temperature"], -1) if case["tail"] else None
    state["row_weight"] = (torch.rand(rows, generator=g, device="cuda") < 0.8).float() * (1.0 / rows) * 64 if case["weights"] else None
    return state


# ---------------------------------------------------------------------------------------- plain forms
def _plain_top(s):
    x = s["logits"].float()
    peak = x.amax(-1, keepdim=True)
    peak = torch.where(peak == -math.inf, 0.0, peak)
    lse = ((x - peak) / s["temperature"]).exp().sum(-1, dtype=torch.float64).log() + peak[:, 0].double() / s["temperature"]
    idx = _top_of(x, s["k"])
    values = x.gather(1, idx)
    idx = torch.where(values == -math.inf, -1, idx)
    return {"idx": idx.to(torch.int32), "values": values, "lse": lse.float()}


def _plain_distill(s):
    tau = s["temperature"]
    z = s["logits"].float()
    rows, vocab = z.shape
    peak = z.amax(-1, keepdim=True)
    e = ((z - peak) / tau).exp()
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    at = s["teacher_idx"].long()
    w = s["row_weight"].double() if s["row_weight"] is not None else torch.ones(rows, dtype=torch.float64, device=z.device)
    logs = (z.gather(1, at) - peak).double() / tau - total.log()   # log s of the teacher's tokens
    v = s["teacher_logits"].double() / tau
    logt = v - (s["teacher_lse"].double()[:, None] if s["teacher_lse"] is not None else torch.logsumexp(v, -1, keepdim=True))
    t = logt.exp()
    loss = (t * (logt - logs)).sum(-1)
    share = e.new_tensor(0.0).double().expand(rows, 1)
    if s["teacher_lse"] is not None:
        rest = e.scatter(1, at, 0.0)
        mass = rest.sum(-1, keepdim=True, dtype=torch.float64)
        share = torch.where(mass > 0, (1 - t.sum(-1, keepdim=True)).clamp(min=0), 0.0)
        loss = loss + torch.where(share > 0, share * (share.log() - (mass / total).log()), 0.0)[:, 0]
    out = {"loss": (w * tau * tau * loss).float()}
    if s["grad"]:
        grad = e * ((t.sum(-1, keepdim=True) + share) / total).float()
        if s["teacher_lse"] is not None:
            grad = grad - rest * torch.where(mass > 0, share / mass, 0.0).float()
        grad.scatter_add_(1, at, -t.float())
        out["dlogits"] = (grad * (w * tau).float()[:, None]).to(s["logits"].dtype)
    return out


def _softmax64(logits, tau):
    x = logits.double()
    e = ((x - x.amax(-1, keepdim=True)) / tau).exp()
    return e / e.sum(-1, keepdim=True)


def _plain_verify(s):
    batch, drafts, tau = s["batch"], s["drafts"], s["temperature"]
    p = _softmax64(s["target"], tau)
    x = s["tokens"].long()
    n = s["n_draft"].long() if s["n_draft"] is not None else torch.full((batch,), drafts, device=x.device)
    px = p[:, :drafts].gather(2, x[:, :, None])[:, :, 0]
    if s["draft"] is not None:
        q = _softmax64(s["draft"], tau)
        qx = q.gather(2, x[:, :, None])[:, :, 0]
    else:
        qx = torch.ones_like(px)
    place = torch.arange(drafts, device=x.device)
    taken = ((s["u_accept"].double() * qx < px) & (place < n[:, None])).long().cumprod(1)
    a = taken.sum(1)
    rows = torch.arange(batch, device=x.device)
    r = p[rows, a]
    if drafts:
        at = a.clamp(max=drafts - 1)
        if s["draft"] is not None:
            there = q[rows, at]
        else:
            there = torch.zeros_like(r).scatter(1, x[rows, at][:, None], 1.0)
        left = (r - torch.where((a < n)[:, None], there, 0.0)).clamp(min=0)
        r = torch.where(left.sum(-1, keepdim=True) > 0, left, r)
    c = r.cumsum(-1)
    token = (c <= s["u_sample"].double()[:, None] * c[:, -1:]).sum(-1)
    place = torch.arange(drafts + 1, device=x.device)
    padded = torch.cat([x, torch.zeros(batch, 1, dtype=torch.long, device=x.device)], 1)
    tokens = torch.where(place < a[:, None], padded, torch.where(place == a[:, None], token[:, None], -1))
    logp = p.gather(2, tokens.clamp(min=0)[:, :, None])[:, :, 0].log()
    return {"tokens": tokens.to(torch.int32), "accepted": a.to(torch.int32), "logprobs": torch.where(place <= a[:, None], logp, 0.0).float()}


def run(state):
    s = state
    if own:
        from cleanba_amd import tokens
        if s["op"] == "top":
            idx, values, lse = tokens.top_logits(s["ctx"], s["logits"], s["k"], temperature=s["temperature"])
            return {"idx": idx, "values": values, "lse": lse}
        if s["op"] == "distill":
            loss, dlogits = tokens.distill_loss_grad(s["ctx"], s["logits"], s["teacher_idx"], s["teacher_logits"], teacher_lse=s["teacher_lse"],
                                                     row_weight=s["row_weight"], temperature=s["temperature"], want_grad=s["grad"])
            return {"loss": loss, "dlogits": dlogits} if s["grad"] else {"loss": loss}
        out, accepted, logprobs = tokens.verify_drafts(s["ctx"], s["target"], s["tokens"], s["u_accept"], s["u_sample"], draft_logits=s["draft"],
                                                       n_draft=s["n_draft"], temperature=s["temperature"])
        return {"tokens": out, "accepted": accepted, "logprobs": logprobs}
    return {"top": _plain_top, "distill": _plain_distill, "verify": _plain_verify}[s["op"]](s)


# ---------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "verify":
        # every row of the drafted positions once (half of them where lengths are drawn), two numbers a draft and one a sequence in, three words a position out
        rows = case["batch"] * (case["drafts"] * (2 if case["draft_logits"] else 1) * (0.5 if case["ragged"] else 1.0) + 1)
        return {"bytes": rows * case["vocab"] * SIZE[case["dtype"]] + case["batch"] * (20 * case["drafts"] + 24), "flops": 4.0 * rows * case["vocab"]}
    logits = case["rows"] * case["vocab"]
    if case["op"] == "top":
        return {"bytes": logits * SIZE[case["dtype"]] + case["rows"] * (8 * case["k"] + 4), "flops": 4.0 * logits}
    grad = bool(case["grad"])
    return {"bytes": logits * SIZE[case["dtype"]] * (1 + grad) + case["rows"] * (8 * case["k"] + 12), "flops": (4.0 + 3.0 * grad) * logits}


# ---------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"top": _exact_top, "distill": _exact_distill, "verify": _exact_verify}[case["op"]](s)


def _row_blocks(rows, vocab):
    step = max(1, (1 << 26) // vocab)
    return [(i, min(rows, i + step)) for i in range(0, rows, step)]


def _exact_top(s):
    parts = []
    for lo, hi in _row_blocks(s["rows"], s["vocab"]):
        x = s["logits"][lo:hi].double()
        best, idx = torch.sort(x, dim=-1, descending=True, stable=True)
        best, idx = best[:, :s["k"]], idx[:, :s["k"]]
        parts.append((idx.masked_fill(best == -math.inf, -1).to(torch.int32), best.clone(), torch.logsumexp(x / s["temperature"], -1)))
    idx, values, lse = (torch.cat(p) for p in zip(*parts))
    return {"idx": idx, "values": values, "lse": lse}


def _exact_distill(s):
    """Loss as a cross-entropy minus an entropy over the teacher's classes; gradient as weighted softmax differences, class by class."""
    tau = s["temperature"]
    losses, grads = [], []
    for lo, hi in _row_blocks(s["rows"], s["vocab"]):
        x = s["logits"][lo:hi].double() / tau
        log_s = torch.log_softmax(x, -1)
        at = s["teacher_idx"][lo:hi].long()
        v = s["teacher_logits"][lo:hi].double() / tau
        in_top = torch.zeros_like(x, dtype=torch.bool).scatter_(1, at, True)
        if s["teacher_lse"] is None:
            t = torch.softmax(v, -1)
            t_rest = torch.zeros_like(t[:, :1])
        else:
            t = torch.exp(v - s["teacher_lse"][lo:hi, None].double())
            t_rest = torch.clamp(1 - t.sum(-1, keepdim=True), min=0)
            t_rest = torch.where(in_top.all(-1, keepdim=True), torch.zeros_like(t_rest), t_rest)
        log_rest = torch.logsumexp(log_s.masked_fill(in_top, -math.inf), -1, keepdim=True)
        entropy = -(torch.special.xlogy(t, t).sum(-1) + torch.special.xlogy(t_rest, t_rest)[:, 0])
        cross = -(t * log_s.gather(1, at)).sum(-1) - torch.where(t_rest > 0, t_rest * log_rest, torch.zeros_like(t_rest))[:, 0]
        w = s["row_weight"][lo:hi].double() if s["row_weight"] is not None else torch.ones_like(cross)
        losses.append(w * tau ** 2 * (cross - entropy))
        if s["grad"]:
            want = torch.zeros_like(x).scatter_add_(1, at, t)
            want += torch.where(in_top | (t_rest <= 0), torch.zeros_like(x), t_rest * torch.exp(log_s - log_rest))
            grads.append((w * tau)[:, None] * (log_s.exp() * (t.sum(-1, keepdim=True) + t_rest) - want))
            if s["logits"].dtype != torch.float32:
                grads[-1] = grads[-1].float()   # (what is compared is held in 16 bits: 32 are exact enough,)
    return {"loss": torch.cat(losses), "dlogits": torch.cat(grads)} if s["grad"] else {"loss": torch.cat(losses)}


def _exact_verify(s):
    """Sequence by sequence, position by position, as the rule is told."""
    drafts, tau = s["drafts"], s["temperature"]
    n = s["n_draft"].tolist() if s["n_draft"] is not None else [drafts] * s["batch"]
    given, u_accept, u_sample = s["tokens"].tolist(), s["u_accept"].tolist(), s["u_sample"].tolist()
    tokens, accepted, logprobs = [], [], []
    for b in range(s["batch"]):
        log_p = torch.log_softmax(s["target"][b].double() / tau, -1)
        out, logs, left = [], [], None
        for i in range(n[b]):
            x = given[b][i]
            p = log_p[i].exp()
            q = torch.softmax(s["draft"][b, i].double() / tau, -1) if s["draft"] is not None else torch.nn.functional.one_hot(torch.tensor(x, device=p.device), p.numel()).double()
            px, qx = torch.stack([p[x], q[x]]).tolist()
            if u_accept[b][i] * qx < px:
                out.append(x)
                continue
            left = torch.relu(p - q)
            left = left if float(left.sum()) > 0 else p
            break
        a = len(out)
        left = log_p[a].exp() if left is None else left
        c = left.cumsum(0)
        out.append(int(torch.searchsorted(c, u_sample[b] * c[-1:], right=True)))
        logs = log_p[torch.arange(a + 1, device=log_p.device), torch.tensor(out, device=log_p.device)].tolist()
        tokens.append(out + [-1] * (drafts - a))
        logprobs.append(logs + [0.0] * (drafts - a))
        accepted.append(a)
    dev = s["target"].device
    return {"tokens": torch.tensor(tokens, dtype=torch.int32, device=dev), "accepted": torch.tensor(accepted, dtype=torch.int32, device=dev),
            "logprobs": torch.tensor(logprobs, dtype=torch.float64, device=dev)}
