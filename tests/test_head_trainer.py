"""lora_ce_score and lora_ce_distill_step: the operators of include/lora_head.h on
a trainer's weight and adapter.

What they share with lora_head_score and lora_head_distill (tested against 64 bits
in test_head.py) has to come out equal bit for bit, the adapter's layout being the
only difference; a distillation step is then lora_head_distill's sums put through
lora_ce_apply_grads."""
import math

import numpy as np
import pytest

import lora_ce

gpu = pytest.mark.gpu
NAMES = ["lora_ce_score", "lora_ce_score_device", "lora_ce_distill_step",
         "lora_ce_distill_step_device"]


@pytest.mark.parametrize("name", NAMES)
def test_a_null_handle_is_refused(name):
    f = getattr(lora_ce.load_library(), name)
    args = [None] * len(f.argtypes)
    for i, t in enumerate(f.argtypes):
        if t is lora_ce.C.c_int32:
            args[i] = 1
        elif t is lora_ce.C.c_float:
            args[i] = 1.0
    assert f(*args) == -1  # LORA_CE_EINVAL


class Pair:
    """A trainer and the same weight, adapter and rows for the stateless calls."""

    def __init__(self, T, V, d, r, seed=0, max_tokens=None, **cfg):
        import torch

        self.torch, self.T, self.V, self.d, self.r = torch, T, V, d, r
        g = np.random.default_rng(1000 * seed + T + V + d + r)
        self.rng = g
        self.W = (g.standard_normal((V, d)) / math.sqrt(d)).astype(np.float16)
        good = g.integers(0, V, T)
        self.H = (g.standard_normal((T, d)) + 8.0 * self.W[good]).astype(np.float32)
        self.A = (g.standard_normal((d, r)) / math.sqrt(d)).astype(np.float32)
        self.B = (g.standard_normal((r, V)) * 0.05).astype(np.float32)
        self.tokens = np.where(g.random(T) < 0.5, good, g.integers(0, V, T)).astype(np.int32)
        self.good = good
        cfg.setdefault("scale", 1.5)
        self.cfg = cfg
        self.m = self.trainer(max_tokens or T)

    def trainer(self, max_tokens):
        m = lora_ce.LoraCE(lora_ce.default_config(self.d, self.V, self.r, max_tokens, **self.cfg))
        m.set_weight(self.W.view(np.uint16))
        m.set_adapter(self.A, self.B)
        return m

    def dev(self, x):
        return self.torch.from_numpy(np.ascontiguousarray(x)).cuda()

    def head(self, A=None, B=None):
        self.dW, self.dA, self.dB = self.dev(self.W), self.dev(self.A if A is None else A), \
            self.dev(self.B if B is None else B)
        return lora_ce.Head(self.dW.data_ptr(), self.dA.data_ptr(), self.dB.data_ptr(), self.d, self.V,
                            self.r, self.cfg["scale"])

    def score(self, k, H=None):
        torch, H = self.torch, self.H if H is None else H
        T, head = H.shape[0], self.head()
        dH, tok = self.dev(H), self.dev(self.tokens[:T])
        out = dict(logprob=torch.zeros(T, device="cuda"), entropy=torch.zeros(T, device="cuda"),
                   top_ids=torch.zeros(T, k, dtype=torch.int32, device="cuda"),
                   top_logprobs=torch.zeros(T, k, device="cuda"))
        ws = torch.empty(lora_ce.head_score_workspace(head, T, k), dtype=torch.uint8, device="cuda")
        lora_ce.head_score(head, dH.data_ptr(), lora_ce.F32, T, tok.data_ptr(), k,
                           *[out[n].data_ptr() if n in ("logprob", "entropy") or k else 0 for n in out],
                           ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return {n: v.cpu().numpy() for n, v in out.items()}

    def lists(self, K):
        g = self.rng
        ids = g.integers(0, self.V, (self.T, K)).astype(np.int32)
        ids[:, 0] = self.good
        ids[g.random((self.T, K)) < 0.1] = -1
        return ids, (g.standard_normal((self.T, K)) + 2.0).astype(np.float32)

    def distill(self, ids, teacher, tau, weight=None, A=None, B=None):
        torch = self.torch
        T, K, head = self.T, ids.shape[1], self.head(A, B)
        dH, i, z = self.dev(self.H), self.dev(ids), self.dev(teacher)
        w = None if weight is None else self.dev(weight)
        loss = torch.zeros(T, device="cuda")
        gA, gB = torch.zeros(self.d, self.r, device="cuda"), torch.zeros(self.r, self.V, device="cuda")
        ws = torch.empty(lora_ce.head_distill_workspace(head, T, K), dtype=torch.uint8, device="cuda")
        lora_ce.head_distill(head, dH.data_ptr(), lora_ce.F32, T, K, i.data_ptr(), z.data_ptr(), tau,
                             0 if w is None else w.data_ptr(), loss.data_ptr(), gA.data_ptr(),
                             gB.data_ptr(), ws.data_ptr(), ws.numel(),
                             torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return loss.cpu().numpy(), gA.cpu().numpy(), gB.cpu().numpy()


@gpu
@pytest.mark.parametrize("T,V,d,r,k", [
    (1, 49152, 576, 4, 5), (9, 20001, 128, 3, 20), (40, 4099, 192, 8, 8), (300, 1000, 576, 16, 4),
    (257, 3000, 64, 20, 0), (1300, 4099, 128, 1, 8), (33, 777, 576, 64, 100),
])
def test_score_is_the_stateless_score(T, V, d, r, k):
    p = Pair(T, V, d, r)
    got, want = p.m.score(p.H, p.tokens, k), p.score(k)
    assert sorted(got) == sorted(n for n in want if k or not n.startswith("top"))
    for n in got:
        np.testing.assert_array_equal(got[n], want[n], err_msg=n)
    only = p.m.score(p.H)
    assert sorted(only) == ["entropy"]
    z = p.H.astype(np.float16).astype(np.float64)
    z = z @ p.W.astype(np.float64).T + 1.5 * ((z @ p.A.astype(np.float64)) @ p.B.astype(np.float64))
    m = z.max(1)
    lse = m + np.log(np.exp(z - m[:, None]).sum(1))
    # sums of at most d / 16 + 12 terms of at most |h| |w| each, 2^-23 apiece
    h, w = np.linalg.norm(p.H, axis=1).max(), np.linalg.norm(p.W.astype(np.float32), axis=1).max()
    tol = (d / 16 + 12) * 2.0**-23 * h * w + 2.0**-19
    assert np.abs(got["logprob"] - (z[np.arange(T), p.tokens] - lse)).max() <= tol


@gpu
def test_score_of_device_buffers_on_the_trainer_stream():
    p = Pair(70, 4099, 128, 4)
    torch = p.torch
    dH, tok = p.dev(p.H), p.dev(p.tokens)
    lp, top = torch.zeros(70, device="cuda"), torch.zeros(70, 6, device="cuda")
    ids = torch.zeros(70, 6, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    p.m.score_device(dH.data_ptr(), lora_ce.F32, 70, tok.data_ptr(), 6, lp.data_ptr(), 0, ids.data_ptr(),
                     top.data_ptr())
    p.m.sync()
    want = p.score(6)
    np.testing.assert_array_equal(lp.cpu().numpy(), want["logprob"])
    np.testing.assert_array_equal(ids.cpu().numpy(), want["top_ids"])
    np.testing.assert_array_equal(top.cpu().numpy(), want["top_logprobs"])


@gpu
@pytest.mark.parametrize("T,V,d,r,K,tau", [
    (1, 4099, 576, 4, 8, 1.0), (300, 4099, 128, 3, 20, 2.0), (257, 1000, 192, 8, 64, 1.0),
    (129, 20001, 64, 16, 5, 0.5), (130, 3000, 576, 33, 16, 2.0), (513, 777, 64, 64, 10, 1.0),
])
@pytest.mark.parametrize("clip", [0.0, 0.1])
def test_distill_step_applies_the_stateless_gradients(T, V, d, r, K, tau, clip):
    p = Pair(T, V, d, r, lr=1e-3, weight_decay=0.01, clip_norm=clip)
    q = p.trainer(T)
    A, B = p.A, p.B
    for step in range(3):
        ids, z = p.lists(K)
        w = None if step == 0 else (p.rng.random(T) * (p.rng.random(T) < 0.8)).astype(np.float32)
        loss = p.m.distill_step(p.H, ids, z, tau, w)
        loss_t, gA, gB = p.distill(ids, z, tau, w, A, B)
        counted = (ids >= 0).any(1) & (True if w is None else w != 0)
        n = max(int(counted.sum()), 1)
        q.apply_grads(gA, gB, n)
        np.testing.assert_array_equal(p.m.token_loss(T), loss_t)
        assert abs(loss - loss_t.astype(np.float64).sum() / n) <= 2.0**-22 * np.abs(loss_t).sum() / n
        mA, mB, loss_sum, n_pred = p.m.get_grads()
        assert n_pred == n and abs(loss_sum / n - loss) <= 2.0**-22 * abs(loss)
        got, want = p.m.get_adapter(), q.get_adapter()
        assert got[2] == want[2] == step + 1
        np.testing.assert_array_equal(got[0], want[0])
        np.testing.assert_array_equal(got[1], want[1])
        A, B = got[0], got[1]
        if clip == 0.0:  # the mean's one rounding
            np.testing.assert_allclose(mA, gA / np.float32(n), rtol=2.0**-22, atol=1e-38)
            np.testing.assert_allclose(mB, gB / np.float32(n), rtol=2.0**-22, atol=1e-38)


@gpu
@pytest.mark.parametrize("r", [4, 16])
def test_distill_step_of_device_buffers(r):
    p = Pair(200, 3000, 128, r)
    q = p.trainer(200)
    ids, z = p.lists(12)
    dH, i, t = p.dev(p.H), p.dev(ids), p.dev(z)
    loss = p.torch.zeros(1, device="cuda")
    p.torch.cuda.synchronize()
    p.m.distill_step_device(dH.data_ptr(), lora_ce.F32, 200, 12, i.data_ptr(), t.data_ptr(), 2.0, 0,
                            loss.data_ptr())
    p.m.distill_step_device(dH.data_ptr(), lora_ce.F32, 200, 12, i.data_ptr(), t.data_ptr(), 2.0)
    p.m.sync()
    first = q.distill_step(p.H, ids, z, 2.0)
    q.distill_step(p.H, ids, z, 2.0)
    assert float(loss) == np.float32(first)
    for a, b in zip(p.m.get_adapter(), q.get_adapter()):
        np.testing.assert_array_equal(a, b)


@gpu
def test_nothing_counted_leaves_a_fresh_adapter():
    p = Pair(40, 1000, 64, 4)
    ids, z = p.lists(4)
    assert p.m.distill_step(p.H, ids, z, 1.0, np.zeros(40, np.float32)) == 0.0
    assert p.m.distill_step(p.H, np.full_like(ids, -1), z) == 0.0
    A, B, step = p.m.get_adapter()
    np.testing.assert_array_equal(A, p.A)
    np.testing.assert_array_equal(B, p.B)
    assert step == 2


@gpu
@pytest.mark.parametrize("r", [4, 32])
def test_scores_and_steps_in_any_order(r):
    """Scores between training steps read the adapter as it stands and leave the
    steps what they were; workspaces grow and serve smaller calls."""
    p = Pair(300, 4099, 128, r, lr=1e-2)
    q = p.trainer(300)
    targets = p.tokens
    ids, z = p.lists(16)
    for m, scores in ((p.m, True), (q, False)):
        for step in range(2):
            if scores:
                m.score(p.H[:5], p.tokens[:5], 8)
            m.step(p.H, targets)
            if scores:
                p.A, p.B = m.get_adapter()[:2]
                got, want = m.score(p.H, p.tokens, 8), p.score(8)
                for n in want:
                    np.testing.assert_array_equal(got[n], want[n], err_msg=n)
            m.distill_step(p.H, ids, z, 2.0)
            if scores:
                m.score(p.H[:1], p.tokens[:1], 128)
            m.step(p.H[:100], targets[:100])
    for a, b in zip(p.m.get_adapter(), q.get_adapter()):
        np.testing.assert_array_equal(a, b)


@gpu
def test_one_entry_is_the_cross_entropy_step():
    """A list of one token is a one-hot teacher: the loss and gradients of
    lora_ce_step, up to the two passes' sums (n 2^-23 |h| |w|)."""
    p = Pair(200, 3000, 128, 8)
    q = p.trainer(200)
    # lora_ce_step predicts row t's target; every row counts
    a = p.m.distill_step(p.H, p.tokens[:, None], np.zeros((200, 1), np.float32))
    b = q.step(p.H, p.tokens)
    h, w = np.linalg.norm(p.H, axis=1).max(), np.linalg.norm(p.W.astype(np.float32), axis=1).max()
    tol = (p.d / 16 + 3) * 2.0**-23 * h * w * 2 + 2.0**-18
    assert abs(a - b) <= tol
    for x, y in zip(p.m.get_grads()[:2], q.get_grads()[:2]):
        assert np.linalg.norm(x - y) <= 2 * tol * np.linalg.norm(y) + 2.0**-14 * np.linalg.norm(y)


@gpu
def test_teacher_scores_feed_the_student_step():
    """The chain as it is used: a teacher's top alternatives are a student's lists;
    the step's loss is the formula's on those lists."""
    p = Pair(150, 2000, 128, 4)
    teacher = Pair(150, 2000, 128, 4, seed=5)
    teacher.m.set_adapter(p.A * 1.5, p.B)
    top = teacher.m.score(p.H, None, 16)
    loss = p.m.distill_step(p.H, top["top_ids"], top["top_logprobs"], 2.0)
    z = p.H.astype(np.float16).astype(np.float64)
    z = z @ p.W.astype(np.float64).T + 1.5 * ((z @ p.A.astype(np.float64)) @ p.B.astype(np.float64))
    z /= 2.0
    lse = np.log(np.exp(z - z.max(1, keepdims=True)).sum(1, keepdims=True)) + z.max(1, keepdims=True)
    t = top["top_logprobs"].astype(np.float64) / 2.0
    lq = t - np.log(np.exp(t).sum(1, keepdims=True))
    want = 4.0 * (np.exp(lq) * (lq - np.take_along_axis(z - lse, top["top_ids"].astype(int), 1))).sum(1).mean()
    h, w = np.linalg.norm(p.H, axis=1).max(), np.linalg.norm(p.W.astype(np.float32), axis=1).max()
    tol = 4.0 * ((p.d / 16 + 1) * 2.0**-23 * h * w + 2.0**-19)
    assert abs(loss - want) <= tol


@gpu
@pytest.mark.parametrize("kw,match", [
    (dict(ids=3000), "token id"), (dict(teacher=math.nan), "teacher logit"),
    (dict(teacher=math.inf), "teacher logit"), (dict(weight=math.nan), "weight"),
    (dict(weight=math.inf), "weight"), (dict(tau=0.0), "temperature"),
])
def test_inputs_that_would_poison_the_adapter_are_refused(kw, match):
    p = Pair(20, 3000, 64, 4)
    ids, z = p.lists(4)
    ids[7, 2] = 1
    w = np.ones(20, np.float32)
    ids[7, 2] = kw.get("ids", 1)
    z[7, 2] = kw.get("teacher", 0.0)
    w[7] = kw.get("weight", 1.0)
    with pytest.raises(lora_ce.LoraCEError, match=match):
        p.m.distill_step(p.H, ids, z, kw.get("tau", 1.0), w)
    A, B, step = p.m.get_adapter()
    np.testing.assert_array_equal(A, p.A)
    np.testing.assert_array_equal(B, p.B)
    assert step == 0
    if "weight" not in kw and "tau" not in kw:  # in a row that counts nothing they are as good as any
        w[7] = 0.0
        assert math.isfinite(p.m.distill_step(p.H, ids, z, 1.0, w))
        assert all(np.isfinite(x).all() for x in p.m.get_adapter()[:2])


@gpu
def test_sizes_states_and_wide_ranks_are_refused():
    p = Pair(20, 1000, 64, 4)
    ids, z = p.lists(4)
    long_ids, long_z = np.tile(ids, (2, 1)), np.tile(z, (2, 1))
    with pytest.raises(lora_ce.LoraCEError, match="T out of range"):
        p.m.score(np.tile(p.H, (2, 1)))
    with pytest.raises(lora_ce.LoraCEError, match="T out of range"):
        p.m.distill_step(np.tile(p.H, (2, 1)), long_ids, long_z)
    with pytest.raises(lora_ce.LoraCEError, match="top_k"):
        p.m.score(p.H, None, 129)
    with pytest.raises(lora_ce.LoraCEError, match="nothing"):
        p.m.score_device(1 << 20, lora_ce.F32, 20, 0, 0, 0, 0, 0, 0)
    with pytest.raises(lora_ce.LoraCEError, match="go together"):
        p.m.score_device(1 << 20, lora_ce.F32, 20, 1 << 20, 0, 0, 1 << 20, 0, 0)
    with pytest.raises(lora_ce.LoraCEError, match="aligned"):
        p.m.score_device((1 << 20) + 8, lora_ce.F32, 20, 0, 0, 0, 1 << 20, 0, 0)
    with pytest.raises(lora_ce.LoraCEError, match="K must"):
        p.m.distill_step(p.H, np.zeros((20, 129), np.int32), np.zeros((20, 129), np.float32))
    fresh = lora_ce.LoraCE(lora_ce.default_config(64, 1000, 4, 20))
    with pytest.raises(lora_ce.LoraCEError, match="weight"):
        fresh.score(p.H)
    wide = Pair(20, 1000, 128, 96)
    with pytest.raises(lora_ce.LoraCEError, match="rank must"):
        wide.m.score(wide.H)
    with pytest.raises(lora_ce.LoraCEError, match="rank must"):
        wide.m.distill_step(wide.H, *wide.lists(4))
