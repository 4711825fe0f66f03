"""The operators on the LoRA head (include/lora_head.h) against a plain
implementation in 64 bits.

Tolerances.  A logit of the GEMM passes is a sum of n = d / 16 + (rank steps)
accumulations in f32, each off by at most one unit in the last place of a
partial sum, which is at most |h| |w| (times the norms); so logits, and the log
of their sum, are off by at most n 2^-23 |h| |w| (the epilogue's exponent
arithmetic, a few 2^-22, and the rounding of the result, 2^-24 of it, come on
top).  Probabilities are off by that much relatively, and so are, as a share
of the sum of the absolute terms, the gradients; the tests ask it of the
2-norms.  Ids are whole numbers and have to be equal."""
import math
import os
import re

import numpy as np
import pytest

import lora_ce

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
gpu = pytest.mark.gpu


# ------------------------------------------------------------------ no GPU
def test_library_exports_every_declared_symbol():
    src = open(os.path.join(REPO, "include", "lora_head.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    names = sorted(set(re.findall(r"\b(lora_head_\w+)\s*\(", src)))
    lib = lora_ce.load_library()
    for n in names:
        assert hasattr(lib, n), n
    assert sorted(lora_ce.HEAD_EXPORTS) == names


def _head(**kw):
    f = dict(W=256, A=256, B=256, dim=576, vocab=49152, rank=4, scale=2.0)
    f.update(kw)
    return lora_ce.Head(*[f[k] for k in ("W", "A", "B", "dim", "vocab", "rank", "scale")])


BAD_HEADS = [dict(dim=100), dict(dim=0), dict(dim=704), dict(vocab=0), dict(vocab=(1 << 19) + 1),
             dict(rank=-1), dict(rank=65), dict(scale=float("nan")), dict(scale=float("inf"))]


@pytest.mark.parametrize("kw", BAD_HEADS)
def test_bad_heads_are_refused(kw):
    with pytest.raises(lora_ce.LoraCEError, match="EINVAL"):
        lora_ce.head_score_workspace(_head(**kw), 8, 4)
    with pytest.raises(lora_ce.LoraCEError, match="EINVAL"):
        lora_ce.head_distill_workspace(_head(**kw), 8, 4)
    with pytest.raises(lora_ce.LoraCEError, match="EINVAL"):
        lora_ce.head_score(_head(**kw), 256, 0, 8, 256, 4, 256, 256, 256, 256, 256, 1 << 40)
    with pytest.raises(lora_ce.LoraCEError, match="EINVAL"):
        lora_ce.head_distill(_head(**kw), 256, 0, 8, 4, 256, 256, 1.0, 0, 256, 256, 256, 256, 1 << 40)


@pytest.mark.parametrize("T,k", [(0, 4), (-1, 4), ((1 << 20) + 1, 4), (8, -1), (8, 129)])
def test_bad_score_sizes_are_refused(T, k):
    with pytest.raises(lora_ce.LoraCEError, match="EINVAL"):
        lora_ce.head_score_workspace(_head(), T, k)
    with pytest.raises(lora_ce.LoraCEError, match="EINVAL"):
        lora_ce.head_score(_head(), 256, 0, T, 256, k, 256, 256, 256, 256, 256, 1 << 40)


def test_more_alternatives_than_tokens_are_refused():
    with pytest.raises(lora_ce.LoraCEError, match="top_k"):
        lora_ce.head_score_workspace(_head(vocab=5), 8, 6)
    assert lora_ce.head_score_workspace(_head(vocab=5), 8, 5) > 0


SCORE = dict(H=256, dtype=0, T=8, tokens=256, k=4, logprob=256, entropy=256, ids=256, lps=256, ws=256,
             n=1 << 40)


@pytest.mark.parametrize("kw,match", [
    (dict(H=0), "H is null"), (dict(H=264), "H must be 16-byte aligned"),
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"),
    (dict(tokens=0), "go together"), (dict(logprob=0), "go together"),
    (dict(tokens=258), "tokens must be 4-byte aligned"),
    (dict(ids=0), "top_ids is null"), (dict(lps=0), "top_logprobs is null"),
    (dict(ws=0), "workspace is null"), (dict(ws=128), "workspace must be 256-byte aligned"),
    (dict(n=1000), "workspace too small"),
    (dict(tokens=0, logprob=0, entropy=0, k=0, ids=0, lps=0), "nothing"),
])
def test_bad_score_arguments_are_refused(kw, match):
    a = dict(SCORE)
    a.update(kw)
    with pytest.raises(lora_ce.LoraCEError, match=match):
        lora_ce.head_score(_head(), a["H"], a["dtype"], a["T"], a["tokens"], a["k"], a["logprob"],
                           a["entropy"], a["ids"], a["lps"], a["ws"], a["n"])


@pytest.mark.parametrize("kw", [dict(W=0), dict(W=264), dict(A=0), dict(B=0)])
def test_bad_head_pointers_are_refused(kw):
    with pytest.raises(lora_ce.LoraCEError, match="EINVAL"):
        lora_ce.head_score(_head(**kw), 256, 0, 8, 256, 4, 256, 256, 256, 256, 256, 1 << 40)


DISTILL = dict(H=256, dtype=0, T=8, K=4, ids=256, teacher=256, tau=1.0, weight=0, loss=256, gA=256,
               gB=256, ws=256, n=1 << 40)


@pytest.mark.parametrize("kw,match", [
    (dict(K=0), "K must"), (dict(K=129), "K must"), (dict(T=0), "T must"),
    (dict(tau=0.0), "temperature"), (dict(tau=-1.0), "temperature"),
    (dict(tau=float("nan")), "temperature"), (dict(tau=101.0), "temperature"),
    (dict(gA=0), "go together"), (dict(gB=0), "go together"),
    (dict(ids=0), "ids is null"), (dict(teacher=0), "teacher is null"),
    (dict(loss=0), "loss is null"), (dict(weight=2), "weight must"),
    (dict(n=1000), "workspace too small"), (dict(dtype=7), "dtype"),
])
def test_bad_distill_arguments_are_refused(kw, match):
    a = dict(DISTILL)
    a.update(kw)
    with pytest.raises(lora_ce.LoraCEError, match=match):
        lora_ce.head_distill(_head(), a["H"], a["dtype"], a["T"], a["K"], a["ids"], a["teacher"],
                             a["tau"], a["weight"], a["loss"], a["gA"], a["gB"], a["ws"], a["n"])


def test_gradients_of_the_base_model_are_refused():
    with pytest.raises(lora_ce.LoraCEError, match="rank of at least 1"):
        lora_ce.head_distill_workspace(_head(rank=0), 8, 4)
    assert lora_ce.head_distill_workspace(_head(rank=0), 8, 4, grads=False) > 0


def test_workspace_grows_with_positions_and_needs_no_logits():
    sizes = [lora_ce.head_score_workspace(_head(), T, 8) for T in (1, 255, 256, 8192, 1 << 20)]
    assert sizes == sorted(sizes)
    assert lora_ce.head_score_workspace(_head(), 8192, 8) < 8192 * 49152  # a quarter of f32 logits
    assert lora_ce.head_distill_workspace(_head(), 8192, 64) < 8192 * 49152


# ------------------------------------------------------------------ on the GPU
DT = {"bf16": lora_ce.BF16, "f16": lora_ce.F16, "f32": lora_ce.F32}


class Problem:
    """Seeded head and hidden states: about unit background logits, a few large
    ones per row."""

    def __init__(self, T, V, d, r, dtype="bf16", seed=0, spread=0.05, boost=10.0):
        import torch

        self.torch, self.T, self.V, self.d, self.r, self.dtype = torch, T, V, d, r, dtype
        g = torch.Generator(device="cuda").manual_seed(1000 * seed + T + V + d + r)
        n = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        u = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
        self.n, self.u = n, u
        self.W = (n(V, d) / math.sqrt(d)).half()
        self.good = (u(T, 4) * V).long().clamp_(0, V - 1)
        H = n(T, d)
        for j in range(4):
            H = H + (boost - 2.0 * j) * u(T, 1) * self.W[self.good[:, j]].float()
        self.H = H.to({"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[dtype])
        self.A, self.B = n(d, r) / math.sqrt(d), n(r, V) * spread
        self.scale = 1.5
        self.tokens = torch.where(u(T) < 0.5, self.good[:, 0], (u(T) * V).long().clamp_(0, V - 1)).int()

    def head(self):
        return lora_ce.Head(self.W.data_ptr(), self.A.data_ptr() if self.r else 0,
                            self.B.data_ptr() if self.r else 0, self.d, self.V, self.r, self.scale)

    def logits(self, A=None, B=None):
        h = self.H.half().double()
        A, B = (self.A if A is None else A).double(), (self.B if B is None else B).double()
        return h @ self.W.double().T + self.scale * ((h @ A) @ B)

    def tol(self):
        """n 2^-23 |h| |w|, see above, and 2^-20 for the epilogue."""
        steps = self.d / 16 + (12 if self.r > 32 else 6 if self.r > 16 else 3 if self.r else 0)
        h, w = self.H.half().float().norm(dim=1).max(), self.W.float().norm(dim=1).max()
        return float(steps * 2.0**-23 * h * w) + 2.0**-20

    def score(self, k, tokens=True, entropy=True, stream=None, ws=None, out=None):
        torch = self.torch
        if out is None:
            out = dict(logprob=torch.full((self.T,), 7.0, device="cuda"),
                       entropy=torch.full((self.T,), 7.0, device="cuda"),
                       ids=torch.full((self.T, k), 7, device="cuda", dtype=torch.int32),
                       lps=torch.full((self.T, k), 7.0, device="cuda"))
        n = lora_ce.head_score_workspace(self.head(), self.T, k)
        if ws is None:
            ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")  # NaNs
        st = (stream or torch.cuda.current_stream()).cuda_stream
        lora_ce.head_score(self.head(), self.H.data_ptr(), DT[self.dtype], self.T,
                           self.tokens.data_ptr() if tokens else 0, k,
                           out["logprob"].data_ptr() if tokens else 0,
                           out["entropy"].data_ptr() if entropy else 0, out["ids"].data_ptr(),
                           out["lps"].data_ptr(), ws.data_ptr(), n, st)
        return out

    def lists(self, K, ragged=True):
        torch = self.torch
        ids = (self.u(self.T, K) * self.V).long().clamp_(0, self.V - 1)
        m = min(K, 4)
        ids[:, :m] = self.good[:, :m]
        teacher = self.n(self.T, K) + 3.0
        if ragged:
            cut = (self.u(self.T) * (K + 1)).long()
            cut = torch.where(self.u(self.T) < 0.3, cut, torch.full_like(cut, K))
            ids[torch.arange(K, device="cuda")[None] >= cut[:, None]] = -1
        self.ids, self.teacher, self.K = ids.int(), teacher, K
        self.weight = None

    def distill(self, tau, grads=True, stream=None, ws=None, out=None):
        torch = self.torch
        if out is None:
            out = dict(loss=torch.full((self.T,), 7.0, device="cuda"),
                       gA=torch.full((self.d, self.r), 7.0, device="cuda"),
                       gB=torch.full((self.r, self.V), 7.0, device="cuda"))
        n = lora_ce.head_distill_workspace(self.head(), self.T, self.K, grads)
        if ws is None:
            ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
        st = (stream or torch.cuda.current_stream()).cuda_stream
        lora_ce.head_distill(self.head(), self.H.data_ptr(), DT[self.dtype], self.T, self.K,
                             self.ids.data_ptr(), self.teacher.data_ptr(), tau,
                             0 if self.weight is None else self.weight.data_ptr(),
                             out["loss"].data_ptr(), out["gA"].data_ptr() if grads else 0,
                             out["gB"].data_ptr() if grads else 0, ws.data_ptr(), n, st)
        return out

    def distill64(self, tau, A=None, B=None, grads=True):
        """loss [T], gA, gB in 64 bits; and the 2-norms that the gradients' terms
        would have without cancelling."""
        torch = self.torch
        w = torch.ones(self.T, dtype=torch.float64, device="cuda") if self.weight is None else self.weight.double()
        ids = self.ids.long()
        ok = ids >= 0
        t = torch.where(ok, self.teacher.double() / tau, torch.full_like(self.teacher, -math.inf).double())
        counted = (t > -math.inf).any(1) & (w != 0)
        t = torch.where(counted[:, None], t, torch.zeros_like(t))
        lq = torch.log_softmax(t, 1)
        q = torch.where(counted[:, None] & ok, lq.exp(), torch.zeros_like(lq))
        H = torch.where(counted[:, None], self.H.half().double(), torch.zeros(1, dtype=torch.float64, device="cuda"))
        A, B = (self.A if A is None else A).double(), (self.B if B is None else B).double()
        U = H @ A
        lp = torch.log_softmax((H @ self.W.double().T + self.scale * (U @ B)) / tau, 1)
        w = torch.where(counted, w, torch.zeros_like(w))
        loss = w * tau**2 * torch.where(q > 0, q * (lq - lp.gather(1, ids.clamp(min=0))), torch.zeros_like(q)).sum(1)
        if not grads:
            return loss
        p = lp.exp()
        target = torch.zeros_like(p).scatter_add_(1, ids.clamp(min=0), q)
        dz, dz_abs = (p - target) * (w * tau)[:, None], (p + target) * (w.abs() * tau)[:, None]
        s = self.scale
        gA, gB = s * (H.T @ (dz @ B.T)), s * (U.T @ dz)
        nA, nB = abs(s) * (H.abs().T @ (dz_abs @ B.abs().T)), abs(s) * (U.abs().T @ dz_abs)
        return loss, gA, gB, float(nA.norm()), float(nB.norm())


def check_score(p, k, out, rows=slice(None)):
    torch = p.torch
    z = p.logits()[rows]
    lse = torch.logsumexp(z, 1, keepdim=True)
    lp = z - lse
    tol = p.tol()
    want = lp.gather(1, p.tokens[rows].long()[:, None])[:, 0]
    assert float((out["logprob"][rows].double() - want).abs().max()) <= tol + 2.0**-24 * float(want.abs().max())
    ent = -(lp.exp() * lp).sum(1)
    # sum p log p: p off by tol relatively, times |log p|
    assert float((out["entropy"][rows].double() - ent).abs().max()) <= tol * (2 + float(ent.max()))
    if k:
        key = torch.sort(lp, dim=1, descending=True, stable=True)
        assert torch.equal(out["ids"][rows].long(), key.indices[:, :k])
        assert float((out["lps"][rows].double() - key.values[:, :k]).abs().max()) <= tol + 2.0**-24 * 32


@gpu
@pytest.mark.parametrize("T,V,d,r,k,dtype", [
    (1, 49152, 576, 4, 5, "bf16"),
    (1, 300, 64, 0, 1, "f16"),
    (2, 1, 64, 1, 1, "f32"),         # one token in the vocabulary
    (7, 63, 64, 2, 63, "bf16"),      # all of a vocabulary smaller than one record
    (24, 65, 128, 3, 20, "f32"),
    (255, 4099, 128, 8, 8, "bf16"),
    (256, 1000, 192, 16, 64, "f16"),
    (257, 3000, 320, 20, 128, "bf16"),
    (129, 2048, 640, 64, 10, "bf16"),  # the widest head: 12 resident K-blocks
    (100, 2048, 640, 13, 10, "f16"),   # 11 resident K-blocks
    (64, 49152, 576, 64, 20, "f32"),
    (1200, 4099, 128, 4, 8, "bf16"),   # a warp per position
    (8, 49152, 576, 16, 20, "bf16"),   # few positions: one, two and four groups of eight
    (9, 49000, 576, 4, 0, "f16"),
    (32, 20001, 128, 33, 50, "f32"),
    (33, 20001, 128, 33, 50, "f32"),   # and one more
    (5, 20035, 640, 64, 8, "bf16"),    # the last block and record cut short
    (3, 100000, 64, 0, 128, "bf16"),
    (1300, 257, 64, 33, 0, "bf16"),    # no alternatives
    (40, 140000, 64, 4, 9, "bf16"),    # a vocabulary larger than the model's
])
def test_score_matches_64_bits(T, V, d, r, k, dtype):
    p = Problem(T, V, d, r, dtype)
    check_score(p, k, p.score(k))


@gpu
def test_score_parts_can_be_left_out():
    p = Problem(33, 1000, 64, 4)
    full, part = p.score(4), p.score(4, tokens=False, entropy=False)
    assert p.torch.equal(full["ids"], part["ids"]) and p.torch.equal(full["lps"], part["lps"])
    assert bool((part["logprob"] == 7).all()) and bool((part["entropy"] == 7).all())
    only = p.score(0)
    tol = p.tol()
    assert float((only["logprob"] - full["logprob"]).abs().max()) <= 2 * tol


@gpu
@pytest.mark.parametrize("T", [9, 1200, 40])
def test_ties_go_to_the_lowest_id(T):
    """Hidden states of zeros (padding): every logit is 0.  And rows of W that
    repeat: their logits are equal to the last bit."""
    torch = pytest.importorskip("torch")
    V, k = 2000, 128
    p = Problem(T, V, 64, 0)
    p.H[::3] = 0
    base = p.W[:50].clone()
    p.W = base[torch.arange(V, device="cuda") % 50].contiguous()  # every row 40 times
    out = p.score(k)
    z = p.logits()
    want = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(out["ids"].long(), want)
    zero = slice(0, None, 3)
    # 2^-23: the rounding of a log of 2000 (7.6) to f32, twice
    assert float((out["entropy"][zero] - math.log(V)).abs().max()) <= 7.6 * 2.0**-23
    p.W = base[:1].expand(V, 64).contiguous()  # every row the same
    out = p.score(k)
    assert torch.equal(out["ids"].long(), torch.arange(k, device="cuda").expand(T, k))


@gpu
def test_near_ties_are_ordered_by_the_exact_logits():
    """Alternatives whose logits differ by less than an f32 sum resolves."""
    torch = pytest.importorskip("torch")
    T, V, d, k = 64, 4096, 576, 20
    p = Problem(T, V, d, 0, "f16")
    # 30 rows of W that differ in one small element only
    ids = torch.arange(30, device="cuda") * 131 + 5
    row = (p.n(d) / math.sqrt(d)).half()
    p.W[ids] = row
    p.W[ids, 0] = (torch.arange(30, device="cuda")[torch.randperm(30, device="cuda")] * 2.0**-24).half()
    p.H = (p.n(T, d) * 0.3 + 12 * row.float()).half()
    z = p.logits()
    want = torch.sort(z, dim=1, descending=True, stable=True)
    assert float((want.values[:, :20] - want.values[:, 1:21]).max()) < 1e-5  # they are near ties
    out = p.score(k)
    assert torch.equal(out["ids"].long(), want.indices[:, :k])


@gpu
@pytest.mark.parametrize("T", [20, 40, 1200])
def test_not_a_number_stays_in_its_row(T):
    torch = pytest.importorskip("torch")
    p = Problem(T, 1000, 64, 4, "f32")
    good = p.score(5)
    p.H[7, 3] = float("nan")
    p.H[9, 0] = float("inf")
    p.H[11, 0] = 1e6  # past f16
    p.tokens[13] = p.V
    p.tokens[14] = -1
    out = p.score(5)
    for t in (7, 9, 11):
        assert math.isnan(float(out["logprob"][t])) and math.isnan(float(out["entropy"][t]))
        assert bool((out["ids"][t] == -1).all()) and bool(out["lps"][t].isnan().all())
    for t in (13, 14):
        assert math.isnan(float(out["logprob"][t]))
        assert torch.equal(out["ids"][t], good["ids"][t])
    rest = torch.ones(T, dtype=torch.bool, device="cuda")
    rest[[7, 9, 11, 13, 14]] = False
    for key in good:
        assert torch.equal(out[key][rest], good[key][rest])


@gpu
@pytest.mark.parametrize("T", [3, 24, 40, 1200])
@pytest.mark.parametrize("v", [0, 500, 4098])
@pytest.mark.parametrize("value", [math.nan, -math.inf])
def test_a_weight_that_is_not_finite_shows(T, v, value):
    """One logit of a row NaN or infinite, in a full tile or the last: the row's
    results are NaN and ids -1, of every row here."""
    p = Problem(T, 4099, 64, 4, "f32")
    p.H[:, 3] = 1.0
    p.W[v, 3] = value
    out = p.score(5)
    assert bool(out["logprob"].isnan().all()) and bool(out["entropy"].isnan().all())
    assert bool((out["ids"] == -1).all()) and bool(out["lps"].isnan().all())
    if math.isnan(value):
        p.lists(6, ragged=False)
        d = p.distill(1.0)
        assert bool(d["loss"].isnan().all()) and bool(d["gA"].isnan().all())


@gpu
@pytest.mark.parametrize("r", [4, 16, 33])
@pytest.mark.parametrize("what", ["id", "nan logit", "nan hidden", "nan weight", "no entries"])
def test_bad_rows_among_few_positions(r, what):
    torch = pytest.importorskip("torch")
    T, V, d, K = 15, 500, 64, 4
    p = Problem(T, V, d, r, "f32")
    p.lists(K, ragged=False)
    p.weight = torch.ones(T, device="cuda")
    good = p.distill(1.0)
    if what == "id":
        p.ids[7, 2] = V
    elif what == "nan logit":
        p.teacher[7, 1] = math.nan
    elif what == "nan hidden":
        p.H[7, 5] = math.nan
    elif what == "nan weight":
        p.weight[7] = math.nan
    else:
        p.ids[7] = -1
        p.H[7] = math.nan
    out = p.distill(1.0)
    rest = torch.arange(T, device="cuda") != 7
    assert torch.equal(out["loss"][rest], good["loss"][rest])
    if what == "no entries":
        assert float(out["loss"][7]) == 0 and bool(out["gB"].isfinite().all())
        p.weight[7] = 0
        p.ids[7] = V + 9
        again = p.distill(1.0)
        assert all(torch.equal(out[k], again[k]) for k in out)
    else:
        assert math.isnan(float(out["loss"][7]))
        assert bool(out["gA"].isnan().all()) and bool(out["gB"].isnan().all())


@gpu
def test_the_first_call_of_a_process_can_be_captured():
    """Kernels load, limits are asked for and set inside a capture as well."""
    import subprocess
    import sys

    code = """
import sys; sys.path[:0] = [%r, %r]
import torch, test_head
out = {}
for T in (5, 300):
    p = test_head.Problem(T, 1000, 64, 16)
    p.lists(6)
    p.weight = p.u(T)
    s = dict(logprob=torch.zeros(T, device="cuda"), entropy=torch.zeros(T, device="cuda"),
             ids=torch.zeros(T, 4, device="cuda", dtype=torch.int32), lps=torch.zeros(T, 4, device="cuda"))
    d = dict(loss=torch.zeros(T, device="cuda"), gA=torch.zeros(64, 16, device="cuda"),
             gB=torch.zeros(16, 1000, device="cuda"))
    w = torch.empty(1 << 26, dtype=torch.uint8, device="cuda")
    st = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        p.score(4, stream=st, ws=w, out=s)
        p.distill(1.5, stream=st, ws=w, out=d)
    g.replay()
    torch.cuda.synchronize()
    a, b = p.score(4), p.distill(1.5)
    assert all(torch.equal(a[k], s[k]) for k in a), T
    assert all(torch.equal(b[k], d[k]) for k in b), T
print("captured")
""" % (os.path.dirname(os.path.abspath(lora_ce.__file__)), os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@gpu
def test_given_buffers_are_written_and_no_more():
    torch = pytest.importorskip("torch")
    T, V, d, r, k = 50, 1000, 64, 5, 6
    p = Problem(T, V, d, r)
    pad = lambda n, dt=torch.float32: torch.full((n + 64,), 77, device="cuda", dtype=dt)  # noqa: E731
    out = dict(logprob=pad(T), entropy=pad(T), ids=pad(T * k, torch.int32), lps=pad(T * k))
    n = lora_ce.head_score_workspace(p.head(), T, k)
    ws = torch.full((n + 256,), 99, dtype=torch.uint8, device="cuda")
    p.score(k, out=out, ws=ws)
    for key, m in (("logprob", T), ("entropy", T), ("ids", T * k), ("lps", T * k)):
        assert bool((out[key][m:] == 77).all()), key
    assert bool((ws[n:] == 99).all())
    p.lists(4)
    out = dict(loss=pad(T), gA=pad(d * r), gB=pad(r * V))
    n = lora_ce.head_distill_workspace(p.head(), T, 4)
    ws = torch.full((n + 256,), 99, dtype=torch.uint8, device="cuda")
    p.distill(1.0, out=out, ws=ws)
    for key, m in (("loss", T), ("gA", d * r), ("gB", r * V)):
        assert bool((out[key][m:] == 77).all()), key
        assert bool((out[key][:m] != 77).all()), key
    assert bool((ws[n:] == 99).all())


def check_distill(p, tau, grads=True):
    torch = p.torch
    out = p.distill(tau, grads)
    tol = p.tol() / tau + 2.0**-20
    want = p.distill64(tau, grads=grads)
    loss = want[0] if grads else want
    w = 1.0 if p.weight is None else float(p.weight.abs().max())
    # log p off by tol; the loss is a difference of numbers of the size of lse
    assert float((out["loss"].double() - loss).abs().max()) <= w * tau**2 * tol * 2 + 2.0**-24 * float(loss.abs().max())
    if grads:
        _, gA, gB, nA, nB = want
        assert bool(torch.isfinite(out["gA"]).all()) and bool(torch.isfinite(out["gB"]).all())
        assert float((out["gA"].double() - gA).norm()) <= tol * nA
        assert float((out["gB"].double() - gB).norm()) <= tol * nB
    return out, want


@gpu
@pytest.mark.parametrize("T,V,d,r,K,tau,dtype", [
    (1, 49152, 576, 4, 8, 1.0, "bf16"),
    (1, 300, 64, 1, 1, 2.0, "f16"),
    (2, 1, 64, 3, 4, 1.0, "f32"),
    (33, 65, 128, 2, 20, 0.5, "bf16"),
    (255, 4099, 128, 8, 128, 2.0, "bf16"),
    (257, 1000, 192, 7, 5, 4.0, "f16"),
    (300, 4099, 128, 16, 33, 1.0, "bf16"),
    (513, 1000, 320, 20, 64, 2.0, "f32"),
    (700, 3000, 192, 64, 10, 1.5, "bf16"),
    (129, 2048, 640, 4, 16, 1.0, "bf16"),   # records not staged
    (129, 2048, 640, 8, 16, 1.0, "bf16"),
    (129, 2048, 640, 64, 16, 1.0, "f16"),   # the widest head
    (200, 2048, 640, 32, 16, 1.0, "f16"),
    (64, 49152, 576, 64, 64, 2.0, "bf16"),
    (2000, 1000, 64, 13, 8, 1.0, "bf16"),
    (3000, 300, 64, 33, 8, 1.0, "bf16"),
])
def test_distill_matches_64_bits(T, V, d, r, K, tau, dtype):
    p = Problem(T, V, d, r, dtype)
    p.lists(K)
    out, _ = check_distill(p, tau)
    p.weight = p.u(T) * 3 - 0.5  # any real weight; some rows 0
    p.weight[p.u(T) < 0.3] = 0
    check_distill(p, tau)
    check_distill(p, tau, grads=False)


@gpu
@pytest.mark.parametrize("T,V,d,r,K,tau,dtype", [
    (1, 300, 64, 0, 4, 1.0, "bf16"), (300, 4099, 128, 0, 64, 2.0, "f16"),
    (129, 2048, 640, 64, 10, 1.0, "bf16"), (129, 2048, 640, 16, 10, 0.7, "f32")])
def test_distill_loss_alone(T, V, d, r, K, tau, dtype):
    p = Problem(T, V, d, r, dtype)
    p.lists(K)
    check_distill(p, tau, grads=False)


@gpu
@pytest.mark.parametrize("T,V,d,r,K,tau,dtype", [
    (1, 4099, 128, 64, 20, 1.0, "f16"),
    (8, 129, 64, 4, 8, 2.0, "bf16"),       # a block of vocabulary rows and one more
    (9, 20001, 576, 16, 64, 1.0, "bf16"),
    (16, 1000, 640, 33, 8, 1.0, "f32"),
    (17, 127, 320, 7, 4, 0.5, "bf16"),
    (32, 49152, 576, 8, 20, 1.5, "f16"),
    (40, 3000, 640, 64, 128, 2.0, "bf16"),
    (47, 2047, 192, 1, 8, 1.0, "f32"),
    (48, 100000, 64, 16, 8, 1.0, "bf16"),
    (49, 4099, 128, 16, 8, 1.0, "bf16"),   # the first of the tensor-core passes
])
@pytest.mark.parametrize("grads", [True, False])
def test_distill_of_few_positions(T, V, d, r, K, tau, dtype, grads):
    p = Problem(T, V, d, r, dtype, seed=2)
    p.lists(K)
    if T % 2 == 0:
        p.weight = p.u(T) * (p.u(T) < 0.7)
    check_distill(p, tau, grads)


@gpu
@pytest.mark.parametrize("r", [4, 8, 16, 64])
@pytest.mark.parametrize("T,V,d,share", [
    (257, 1000, 64, 0.5), (290, 4099, 128, 0.0), (700, 2048, 576, 0.3), (1500, 300, 64, 0.05),
    (3000, 4099, 64, 0.001), (2048, 777, 128, 1.0), (5000, 200, 64, 0.4),
])
def test_masked_positions_anywhere(r, T, V, d, share):
    """Weights of 0 in whole stretches and one by one, over more than one tile of
    positions: the passes leave their tiles out, and what lies there does not
    matter.  None, few, and all of them count; the loss is that of the weights."""
    p = Problem(T, V, d, r, seed=4)
    p.lists(9, ragged=share < 1.0)
    torch = p.torch
    w = 0.5 + 0.5 * p.u(T)
    w = torch.where(p.u(T) < share, w, torch.zeros_like(w))
    if 0.0 < share < 1.0:
        w[: T // 5] = 0.0
        w[T // 2: T // 2 + 3] = 1.0
        tol = p.tol()
        p.tol = lambda: tol  # of the rows as they were
        p.H[w == 0] = math.nan
        p.teacher[w == 0] = math.inf
    p.weight = w
    out, (loss, *_) = check_distill(p, 1.5)
    assert bool((out["loss"][w == 0] == 0).all())
    alone = p.distill(1.5, grads=False)["loss"]
    tol = 1.5**2 * 2 * (p.tol() / 1.5 + 2.0**-20)
    assert float((alone.double() - loss).abs().max()) <= tol + 2.0**-24 * float(loss.abs().max())
    if share == 1.0:  # nothing to leave out: the order is the positions' own
        p.weight = torch.ones_like(w)
        a = p.distill(1.5)
        p.weight = None
        b = p.distill(1.5)
        assert all(torch.equal(a[k], b[k]) for k in a)


@gpu
@pytest.mark.parametrize("r", [4, 8, 16, 64])
def test_gradient_is_the_slope_of_the_loss(r):
    """Central differences of the 64-bit loss along a random direction: the
    truncation error of a step e is e^2 / 6 times a third derivative of order
    of the loss here, so e = 1e-4 leaves 1e-8; what remains is the gradients'
    own tolerance against the sum of the terms' absolute values."""
    T, V, d = 150, 1000, 128
    p = Problem(T, V, d, r)
    p.lists(12)
    p.weight = p.u(T)
    tau, e = 1.7, 1e-4
    out, (_, _, _, nA, nB) = check_distill(p, tau)
    dA, dB = p.n(d, r).double() / math.sqrt(d), p.n(r, V).double() * 0.1
    for D, g, norm in ((dict(A=dA), out["gA"], nA), (dict(B=dB), out["gB"], nB)):
        at = lambda s: float(p.distill64(tau, grads=False, **{  # noqa: E731
            k: getattr(p, k).double() + s * e * v for k, v in D.items()}).sum())
        slope = (at(1) - at(-1)) / (2 * e)
        v = list(D.values())[0]
        got = float((g.double() * v).sum())
        assert abs(got - slope) <= (p.tol() / tau + 2.0**-20) * norm * float(v.norm()) + 1e-5 * abs(slope)


@gpu
@pytest.mark.parametrize("r", [4, 8, 16, 64])
def test_rows_that_count_nothing_hold_anything(r):
    """Weight 0, no entry, entries of -inf alone: loss 0 and no part in the
    gradients, with NaN and infinities in the hidden state, and NaN in the logits
    of absent entries."""
    torch = pytest.importorskip("torch")
    T, V, d, K = 300, 1000, 64, 6
    p = Problem(T, V, d, r, "f32")
    p.lists(K, ragged=False)
    p.weight = torch.ones(T, device="cuda")
    off = torch.zeros(T, dtype=torch.bool, device="cuda")
    off[::5] = off[1::5] = True
    keep = p.H.clone(), p.ids.clone(), p.teacher.clone(), p.weight.clone()
    p.weight[off] = 0
    clean = p.distill(1.5)
    p.weight[1::5] = 1
    p.ids[1::5] = -1                      # rows 1, 6, ..: no entries
    p.ids[::10, 0] = V + 5                # rows 0, 10, ..: weight 0 and a wild id
    p.teacher[1::5] = float("nan")
    p.H[off] = float("nan")
    p.H[::10] = float("inf")
    got = p.distill(1.5)
    for key in clean:
        assert torch.equal(clean[key], got[key]), key
    assert bool((got["loss"][off] == 0).all())
    # entries of -inf weigh nothing; a row of them alone counts nothing
    p.H, p.ids, p.teacher, p.weight = keep
    p.weight = None
    p.teacher[2::7] = -math.inf
    p.teacher[3::7, 1:] = -math.inf
    out, want = check_distill(p, 1.0)
    assert bool((out["loss"][2::7] == 0).all())
    # every row off
    p.ids[:] = -1
    out = p.distill(1.0)
    for key in out:
        assert bool((out[key] == 0).all()), key


@gpu
@pytest.mark.parametrize("r", [4, 16])
@pytest.mark.parametrize("what", ["id", "nan logit", "inf logit", "nan hidden", "nan weight"])
def test_bad_counted_rows_make_the_gradients_nan(r, what):
    torch = pytest.importorskip("torch")
    T, V, d, K = 100, 500, 64, 4
    p = Problem(T, V, d, r, "f32")
    p.lists(K, ragged=False)
    p.weight = torch.ones(T, device="cuda")
    good = p.distill(1.0)["loss"]
    if what == "id":
        p.ids[17, 2] = V
    elif what == "nan logit":
        p.teacher[17, 1] = float("nan")
    elif what == "inf logit":
        p.teacher[17, 1] = float("inf")
    elif what == "nan hidden":
        p.H[17, 5] = float("nan")
    else:
        p.weight[17] = float("nan")
    out = p.distill(1.0)
    assert math.isnan(float(out["loss"][17]))
    rest = torch.arange(T, device="cuda") != 17
    assert torch.equal(out["loss"][rest], good[rest])
    assert bool(out["gA"].isnan().all()) and bool(out["gB"].isnan().all())
    assert math.isnan(float(p.distill(1.0, grads=False)["loss"][17]))


@gpu
@pytest.mark.parametrize("r", [3, 16])
def test_same_id_twice_and_a_fresh_adapter(r):
    torch = pytest.importorskip("torch")
    p = Problem(200, 1000, 64, r)
    p.lists(8, ragged=False)
    p.ids[:, 4:] = p.ids[:, :1]  # one token holds most of the list
    check_distill(p, 1.0)
    p.B.zero_()                  # LoRA's initial B: gA is 0, gB is not
    out, _ = check_distill(p, 2.0)
    assert bool((out["gA"] == 0).all()) and float(out["gB"].abs().max()) > 0


@gpu
@pytest.mark.parametrize("tau", [0.01, 0.1, 100.0])
@pytest.mark.parametrize("r", [4, 32])
def test_temperatures_far_from_one(tau, r):
    p = Problem(130, 1000, 64, r)
    p.lists(8)
    check_distill(p, tau)


@gpu
@pytest.mark.parametrize("r", [4, 8, 16, 64])
def test_weights_of_any_size(r):
    """Gradients scale with the weights: tiny and huge ones lose nothing."""
    torch = pytest.importorskip("torch")
    p = Problem(300, 1000, 64, r)
    p.lists(8)
    p.weight = torch.ones(300, device="cuda")
    one = p.distill(1.0)
    for e in (-40, 30):
        p.weight[:] = 2.0**e
        out = p.distill(1.0)
        for key in one:  # powers of two: the same bits
            assert torch.equal(out[key], one[key] * 2.0**e), (e, key)


@gpu
@pytest.mark.parametrize("r,T", [(4, 300), (16, 129)])
def test_one_entry_is_the_cross_entropy_of_the_step(r, T):
    """K = 1 at temperature 1 against lora_ce_step's gradients (mean over T) on
    the same inputs; the step's own parity tolerance is 1e-3, its arithmetic's
    error some 1e-5."""
    torch = pytest.importorskip("torch")
    V, d = 4099, 128
    p = Problem(T, V, d, r)
    p.ids, p.teacher, p.K, p.weight = p.tokens[:, None].contiguous(), torch.zeros(T, 1, device="cuda"), 1, None
    out, _ = check_distill(p, 1.0)
    m = lora_ce.LoraCE(lora_ce.default_config(d, V, r, T, scale=p.scale))
    m.set_weight(p.W.view(torch.int16).cpu().numpy().view(np.uint16))
    m.set_adapter(p.A.cpu().numpy(), p.B.cpu().numpy(), 0)
    m.step(p.H.view(torch.int16).cpu().numpy().view(np.uint16), p.tokens.cpu().numpy())
    gA, gB, loss_sum, _ = m.get_grads()
    m.close()
    for a, b in ((out["gA"].cpu().numpy() / T, gA), (out["gB"].cpu().numpy() / T, gB)):
        assert np.linalg.norm(a - b) <= 1e-4 * np.linalg.norm(b)
    assert abs(float(out["loss"].double().sum()) - loss_sum) <= 1e-5 * loss_sum


@gpu
@pytest.mark.parametrize("r", [4, 16])
@pytest.mark.parametrize("T", [12, 300, 700])  # few positions; most; masked ones among them
def test_streams_graphs_and_repeats(T, r):
    """The same bits from another stream, from a captured and replayed graph with
    new inputs in its buffers, and from two calls at once."""
    torch = pytest.importorskip("torch")
    p, o = Problem(T, 4099, 128, r), Problem(T, 4099, 128, r, seed=1)
    for x in (p, o):
        x.lists(8)
        x.weight = x.u(T) * (x.u(T) < 0.5) if T == 700 else torch.ones(T, device="cuda")
    first = dict(p.score(8), **p.distill(2.0))
    other = dict(o.score(8), **o.distill(2.0))
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):  # two calls at once, each with its workspace
        with torch.cuda.stream(a):
            x = dict(p.score(8), **p.distill(2.0))
        with torch.cuda.stream(b):
            y = dict(o.score(8), **o.distill(2.0))
        torch.cuda.synchronize()
        for key in first:
            assert torch.equal(x[key], first[key]) and torch.equal(y[key], other[key]), key
    so, do = p.score(8), p.distill(2.0)
    n1 = lora_ce.head_score_workspace(p.head(), p.T, 8)
    n2 = lora_ce.head_distill_workspace(p.head(), p.T, 8)
    ws1 = torch.zeros(n1, dtype=torch.uint8, device="cuda")
    ws2 = torch.zeros(n2, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.score(8, out=so, ws=ws1, stream=torch.cuda.current_stream())
        p.distill(2.0, out=do, ws=ws2, stream=torch.cuda.current_stream())
    for q, want in ((o, other), (p, first), (o, other)):
        keep = {k: getattr(q, k).clone() for k in ("H", "A", "B", "W", "ids", "teacher", "tokens", "weight")}
        for k, v in keep.items():
            getattr(p, k).copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for key, got in dict(so, **do).items():
            assert torch.equal(got, want[key]), key
        if q is p:
            continue
        # p's own inputs come back for the next round
        fresh = Problem(T, 4099, 128, r)
        fresh.lists(8)
        fresh.weight = fresh.u(T) * (fresh.u(T) < 0.5) if T == 700 else torch.ones(T, device="cuda")
        for k in keep:
            getattr(p, k).copy_(getattr(fresh, k))


@gpu
def test_memory_elsewhere_is_refused():
    torch = pytest.importorskip("torch")
    p = Problem(8, 300, 64, 4)
    p.tokens = p.tokens.cpu()
    with pytest.raises(lora_ce.LoraCEError, match="tokens is not memory of the current device"):
        p.score(2)
    p.tokens = p.tokens.pin_memory()
    with pytest.raises(lora_ce.LoraCEError, match="tokens is not memory"):
        p.score(2)
    p.lists(2)
    p.teacher = p.teacher.cpu()
    with pytest.raises(lora_ce.LoraCEError, match="teacher is not memory"):
        p.distill(1.0)
    torch.cuda.synchronize()


@gpu
def test_teacher_to_student():
    """As used: the base model's alternatives are the lists of the student's
    distillation; where the student is the teacher and the lists hold all of the
    vocabulary, loss and gradients vanish."""
    torch = pytest.importorskip("torch")
    p = Problem(300, 100, 64, 4)
    top = p.score(100)
    p.ids, p.teacher, p.K, p.weight = top["ids"], top["lps"], 100, None
    out = p.distill(1.0)
    _, _, _, nA, nB = p.distill64(1.0)
    assert float(out["loss"].abs().max()) <= 2 * p.tol()
    assert float(out["gA"].norm()) <= 2 * p.tol() * nA and float(out["gB"].norm()) <= 2 * p.tol() * nB
    # another student: the loss falls along the negative gradient
    q = Problem(300, 4099, 128, 8)
    top = q.score(16)
    q.ids, q.teacher, q.K, q.weight = top["ids"], top["lps"], 16, None
    q.B.mul_(0.5)
    one = q.distill(2.0)
    want = q.distill64(2.0)
    assert float((one["gB"].double() - want[2]).norm()) <= (q.tol() / 2 + 2.0**-20) * want[4]
