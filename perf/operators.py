"""What is measured of the operators on the LoRA head: h -> logits over the
vocabulary, z = h . W^T + scale * (h . A) . B with h rounded to f16 (as every
entry point of the library reads hidden states), W the tied lm_head [V][d] f16,
A [d][r] and B [r][V] f32.

* "score": per position the log probability of a given token, the entropy of
  the distribution and the top alternatives (ids and log probabilities; ties go
  to the lowest id).
* "distill": per position KL(teacher || student) over the teacher's top
  logits, tau^2 * sum_k q_k (log q_k - log p_k), with q the softmax of the
  teacher's K logits / tau over the entries with an id >= 0 and p the softmax of
  z / tau over the whole vocabulary; times the position's weight; and, unless only
  the loss is wanted, the gradients of the sum over positions in A and B.

`run` computes both in their plain form, or, where `own` is set, through the
library's entry points.
"""
import math

import torch

own = False

_library = None


def _lib():
    global _library
    if _library is None:
        import __graft_entry__
        _library = __graft_entry__.package()[0]
    return _library


MARGIN = 8  # candidates beyond top_k whose logits the plain form computes again in 64 bits


def listed():
    score = dict(op="score", V=49152, d=576)
    distill = dict(op="distill", V=49152, d=576, weighted=False, grads=True, tau=1.0)
    return [
        # one generated token with its five best alternatives: latency
        dict(score, name="score decode 1", T=1, r=4, k=5, dtype="bf16"),
        # a decode batch, an API's usual limit of 20 alternatives
        dict(score, name="score decode 24", T=24, r=16, k=20, dtype="f16"),
        # one sample of the trainer (256 tokens, 255 predictions) scored in one call
        dict(score, name="score sample 255", T=255, r=8, k=8, dtype="bf16"),
        # perplexity over a packed batch: no alternatives wanted
        dict(score, name="score packed 2047", T=2047, r=64, k=0, dtype="bf16"),
        # the teacher side of distillation: the base model's 64 best tokens
        dict(score, name="score teacher 4096", T=4096, r=0, k=64, dtype="bf16"),
        # a large evaluation batch
        dict(score, name="score batch 8192", T=8192, r=4, k=8, dtype="bf16"),
        # a small vocabulary and head, nothing on a tile boundary
        dict(score, name="score small 777", T=777, V=4099, d=128, r=3, k=10, dtype="f32"),
        # one short sample: launches count
        dict(distill, name="distill sample 33", T=33, r=4, K=8, dtype="bf16"),
        # one sample of the trainer, softened
        dict(distill, name="distill sample 255", T=255, r=8, K=20, tau=2.0, dtype="bf16"),
        # validation: the loss alone
        dict(distill, name="distill loss 2047", T=2047, r=16, K=32, tau=2.0, grads=False, dtype="f16"),
        # the isolated step's size
        dict(distill, name="distill step 8192", T=8192, r=4, K=8, dtype="bf16"),
        # a large rank, the whole teacher list, prompt positions masked by weight 0
        dict(distill, name="distill wide 8000", T=8000, r=64, K=64, tau=1.5, weighted=True, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("score", "distill"))
    big = rng.random() < 0.6  # the model's own head, or another of any size
    V = 49152 if big else _log_int(rng, 300, 49152)
    d = 576 if big else 64 * rng.randint(1, 9)
    T = _log_int(rng, 1, 8000)
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op == "score":
        return dict(op=op, T=T, V=V, d=d, r=rng.choice((0, _log_int(rng, 1, 64))), k=rng.choice((0, _log_int(rng, 1, 64))), dtype=dtype)
    return dict(op=op, T=T, V=V, d=d, r=_log_int(rng, 1, 64), K=_log_int(rng, 1, 64), tau=rng.choice((1.0, 1.5, 2.0, 4.0)),
                weighted=rng.random() < 0.5, grads=rng.random() < 0.75, dtype=dtype)


def prepare(case, seed):
    """A head whose weight rows have about unit norm, an adapter that has been
    trained a little, and hidden states that favour a few Zipf-distributed tokens
    each (logits of about 5 to 11 over a background of about unit spread, as of a
    language model between sure and unsure)."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    T, V, d, r = case["T"], case["V"], case["d"], case["r"]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device=dev, generator=g)

    W = (normal(V, d) / math.sqrt(d)).half()
    n_good = 6
    # token ids with p(k) ~ 1 / k, spread over the vocabulary
    good = torch.exp(uniform(T, n_good) * math.log(V)).long().sub_(1).clamp_(0, V - 1)
    boost = (5.0 + 6.0 * uniform(T, 1)) - 1.5 * uniform(T, n_good) * torch.arange(n_good, device=dev)
    H = normal(T, d)
    for j in range(n_good):
        H += boost[:, j : j + 1] * W[good[:, j]].float()
    H = H.to({"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[case["dtype"]])
    A = normal(d, r) / math.sqrt(d)
    B = normal(r, V) * 0.05
    state = dict(case=case, W=W, H=H, A=A, B=B, scale=2.0)
    if case["op"] == "score":
        k = case["k"]
        tokens = torch.where(uniform(T) < 0.6, good[:, 0], (uniform(T) * V).long().clamp_(0, V - 1))
        state.update(tokens=tokens.int(), logprob=torch.empty(T, device=dev), entropy=torch.empty(T, device=dev),
                     top_ids=torch.empty(T, k, device=dev, dtype=torch.int32), top_logprobs=torch.empty(T, k, device=dev))
    else:
        K = case["K"]
        n = min(K, n_good)
        ids = (uniform(T, K) * V).long().clamp_(0, V - 1)
        ids[:, :n] = good[:, :n]
        teacher = normal(T, K) * 0.8 + 2.0
        teacher[:, :n] = boost[:, :n] + 0.5 * normal(T, n)
        # lists cut short where the teacher was sure (every eighth), a few of them empty
        length = torch.where(uniform(T) < 0.125, (uniform(T) * (K + 1)).long(), torch.full((T,), K, device=dev))
        ids[torch.arange(K, device=dev)[None, :] >= length[:, None]] = -1
        state.update(ids=ids.int(), teacher=teacher, weight=None, loss=torch.empty(T, device=dev),
                     gA=torch.empty(d, r, device=dev), gB=torch.empty(r, V, device=dev))
        if case["weighted"]:  # prompt positions count nothing, the answer's by 0.5 to 1
            w = 0.5 + 0.5 * uniform(T)
            state["weight"] = torch.where(uniform(T) < 0.3, torch.zeros_like(w), w)
    return state


# ---------------------------------------------------------------- plain forms
def _logits(s):
    h = s["H"].half().float()
    U = h @ s["A"]
    return h, U, h @ s["W"].float().T + s["scale"] * (U @ s["B"])


def _logits_at(s, ids):
    """The logits of chosen ids [T][n] in 64 bits: they order the alternatives."""
    h = s["H"].half().double()
    sU = s["scale"] * (h @ s["A"].double())
    z = (s["W"][ids].double() @ h[:, :, None])[:, :, 0]
    return z + (s["B"].T[ids].double() @ sU[:, :, None])[:, :, 0]


def _plain_score(s):
    case = s["case"]
    _, _, z = _logits(s)
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    S = e.sum(1)
    lse = m[:, 0] + torch.log(S)
    entropy = torch.log(S) - (e * (z - m)).sum(1) / S
    logprob = (_logits_at(s, s["tokens"].long()[:, None])[:, 0] - lse).float()
    k = case["k"]
    if not k:
        return dict(logprob=logprob, entropy=entropy)
    ids = torch.topk(z, min(k + MARGIN, case["V"]), dim=1).indices.sort(dim=1).values
    zc = _logits_at(s, ids)
    order = torch.sort(zc, dim=1, descending=True, stable=True).indices[:, :k]  # ids ascend: ties go to the lowest
    return dict(logprob=logprob, entropy=entropy, top_ids=ids.gather(1, order).int(),
                top_logprobs=(zc.gather(1, order) - lse[:, None].double()).float())


def _plain_distill(s):
    case, tau = s["case"], s["case"]["tau"]
    h, U, z = _logits(s)
    valid = s["ids"] >= 0
    ids = s["ids"].long().clamp(min=0)
    t = torch.where(valid, s["teacher"] / tau, torch.full_like(s["teacher"], -math.inf))
    some = valid.any(1, keepdim=True)
    top = torch.where(some, t.amax(1, keepdim=True), torch.zeros_like(t[:, :1]))
    q = torch.exp(t - top)
    total = q.sum(1, keepdim=True)
    log_q = t - top - torch.log(torch.where(some, total, torch.ones_like(total)))
    q = torch.exp(log_q)
    y = z / tau
    m = y.amax(1, keepdim=True)
    e = torch.exp(y - m)
    S = e.sum(1, keepdim=True)
    log_p = y.gather(1, ids) - m - torch.log(S)
    w = some[:, 0].float() if s["weight"] is None else s["weight"] * some[:, 0]
    loss = w * tau * tau * torch.where(valid, q * (log_q - log_p), torch.zeros_like(q)).sum(1)
    if not case["grads"]:
        return dict(loss=loss)
    dz = e / S
    dz.scatter_add_(1, ids, -q)
    dz *= (w * tau)[:, None]
    dU = s["scale"] * (dz @ s["B"].T)
    return dict(loss=loss, gA=h.T @ dU, gB=s["scale"] * (U.T @ dz))


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if not own:
        return _plain_score(state) if case["op"] == "score" else _plain_distill(state)
    lib = _lib()
    T, V, d, r = case["T"], case["V"], case["d"], case["r"]
    dtype = {"bf16": lib.BF16, "f16": lib.F16, "f32": lib.F32}[case["dtype"]]
    stream = torch.cuda.current_stream().cuda_stream
    head = lib.Head(state["W"].data_ptr(), state["A"].data_ptr(), state["B"].data_ptr(), d, V, r, state["scale"])
    if case["op"] == "score":
        k = case["k"]
        work = torch.empty(lib.head_score_workspace(head, T, k), dtype=torch.uint8, device="cuda")
        lib.head_score(head, state["H"].data_ptr(), dtype, T, state["tokens"].data_ptr(), k, state["logprob"].data_ptr(),
                       state["entropy"].data_ptr(), state["top_ids"].data_ptr(), state["top_logprobs"].data_ptr(),
                       work.data_ptr(), work.numel(), stream)
        out = dict(logprob=state["logprob"], entropy=state["entropy"])
        return dict(out, top_ids=state["top_ids"], top_logprobs=state["top_logprobs"]) if k else out
    K, grads = case["K"], case["grads"]
    work = torch.empty(lib.head_distill_workspace(head, T, K, grads), dtype=torch.uint8, device="cuda")
    weight = state["weight"]
    lib.head_distill(head, state["H"].data_ptr(), dtype, T, K, state["ids"].data_ptr(), state["teacher"].data_ptr(),
                     case["tau"], 0 if weight is None else weight.data_ptr(), state["loss"].data_ptr(),
                     state["gA"].data_ptr() if grads else 0, state["gB"].data_ptr() if grads else 0,
                     work.data_ptr(), work.numel(), stream)
    return dict(loss=state["loss"], gA=state["gA"], gB=state["gB"]) if grads else dict(loss=state["loss"])


def work(case):
    """Each input read once, each output written once; the products that the
    definition asks for: the logits (h . W^T and the rank term), and for the
    gradients the same again is not counted, only dz against B, U and h."""
    T, V, d, r = case["T"], case["V"], case["d"], case["r"]
    size = 4 if case["dtype"] == "f32" else 2
    data = 2 * V * d + size * T * d + 4 * r * (d + V)
    flops = 2 * T * V * d + 2 * T * r * (d + V)
    if case["op"] == "score":
        return dict(bytes=data + 4 * T + 4 * T * (2 + 2 * case["k"]), flops=flops)
    data += 8 * T * case["K"] + 4 * T * (2 if case["weighted"] else 1)
    if case["grads"]:
        data += 4 * r * (d + V)
        flops += 2 * T * r * (2 * V + d)
    return dict(bytes=data, flops=flops)


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    W, A, B = s["W"].double(), s["A"].double(), s["B"].double()
    T, step, parts = case["T"], 1024, []
    gA, gB = torch.zeros_like(A), torch.zeros_like(B)
    for t0 in range(0, T, step):
        rows = slice(t0, min(T, t0 + step))
        h = s["H"][rows].half().double()
        U = h @ A
        z = torch.addmm(h @ W.T, U, B, alpha=s["scale"])
        if case["op"] == "score":
            lse = torch.logsumexp(z, 1, keepdim=True)
            lp = z - lse
            got = [lp.gather(1, s["tokens"][rows].long()[:, None])[:, 0], -(lp.exp() * lp).sum(1)]
            if case["k"]:
                got += list(torch.topk(lp, case["k"], dim=1))
            parts.append(got)
            continue
        tau, ids = case["tau"], s["ids"][rows].long()
        lp = torch.log_softmax(z / tau, 1)
        del z
        w = torch.ones(len(h), dtype=torch.float64, device=h.device) if s["weight"] is None else s["weight"][rows].double()
        t = s["teacher"][rows].double() / tau
        t[ids < 0] = -math.inf
        lq = t - torch.logsumexp(t, 1, keepdim=True)
        q = torch.nan_to_num(lq.exp(), nan=0.0)  # an empty list: no target at all
        lpk = lp.gather(1, ids.clamp(min=0))
        w = w * (ids >= 0).any(1)
        parts.append([w * tau**2 * torch.where(q > 0, q * (lq - lpk), 0 * q).sum(1)])
        if case["grads"]:
            target = torch.zeros_like(lp).scatter_add_(1, ids.clamp(min=0), q)
            dz = (lp.exp() - target) * (w * tau)[:, None]
            gB += s["scale"] * (U.T @ dz)
            gA += s["scale"] * (h.T @ (dz @ B.T))
    cols = [torch.cat(c) for c in zip(*parts)]
    if case["op"] == "score":
        out = dict(logprob=cols[0], entropy=cols[1])
        return dict(out, top_ids=cols[3].int(), top_logprobs=cols[2]) if case["k"] else out
    return dict(loss=cols[0], gA=gA, gB=gB) if case["grads"] else dict(loss=cols[0])
