"""The operators on the LoRA head (include/lora_head.h) at their edges: ties and
crowds among the alternatives, both sides of every dispatch, ranges of the operands,
sums that cancel, gradients element by element.  The tolerances are those of
test_head.py unless a test derives its own."""
import math

import pytest

from test_head import Problem, check_distill, check_score

gpu = pytest.mark.gpu


class Given(Problem):
    """Logits as given, exactly: z [V] (f16 values) times +-2^n by position."""

    def __init__(self, T, z, d=64, r=0):
        super().__init__(T, len(z), d, r)
        torch = self.torch
        self.W.zero_()
        self.W[:, 0] = z.cuda().half()
        self.H = torch.zeros(T, d, device="cuda", dtype=torch.bfloat16)
        self.H[:, 0] = torch.tensor([1.0, 0.5, -1.0, 2.0], device="cuda")[torch.arange(T, device="cuda") % 4]


def _crowds(V, what):
    import torch
    g = torch.Generator().manual_seed(V)
    z = -4 - 2 * torch.rand(V, generator=g)
    at = V * 13 // 16 // 64 * 64 + 1  # one chunk of eight columns, high up
    if what == "block of ties":
        z[:192] = 0
        z[at:at + 4] = torch.tensor([5.0, 4.5, 4.0, 3.5])
    elif what == "all tied but three":
        z[:] = 0
        z[at:at + 3] = torch.tensor([1.0, 3.0, 2.0])
    elif what == "large ones in few records":
        n = 640
        z[at - 1:at - 1 + n] = (5 + torch.randperm(n, generator=g) / 128)[:len(z[at - 1:at - 1 + n])]
    else:  # more ties than a list holds, above a second crowd
        z[:V // 2] = 1
        z[V // 2:V // 2 + 40] = 2
    return z


@gpu
@pytest.mark.parametrize("T,V,k", [
    (9, 49152, 8),      # few positions
    (100, 49152, 8), (1200, 49152, 8),   # four warps per position, one
    (40, 140000, 8),    # eight
    (9, 49152, 128), (300, 49152, 128),
    (100, 4099, 20), (2400, 4099, 20),   # records of 8 columns
    (30, 600, 100),     # of one
])
@pytest.mark.parametrize("what", ["block of ties", "all tied but three", "large ones in few records",
                                  "two crowds"])
def test_larger_logits_are_not_lost_among_ties(T, V, k, what):
    """Columns that a record does not name come before ties at the k-th place,
    wherever they lie and however many ties there are."""
    p = Given(T, _crowds(V, what))
    check_score(p, k, p.score(k))


@gpu
@pytest.mark.parametrize("r", [3, 8, 16, 64])
@pytest.mark.parametrize("T", [7, 31, 100, 300, 1500])
@pytest.mark.parametrize("weights", [False, True])
def test_rows_whose_entries_are_all_minus_infinity_hold_anything(T, r, weights):
    """Such a row has no entry: loss 0 and no part in the gradients, the same bits
    as with no ids, with NaN and infinities in its hidden state."""
    import torch
    V, K = 1000, 6
    p = Problem(T, V, 64, r, "f32")
    p.lists(K, ragged=False)
    p.weight = torch.where(torch.arange(T, device="cuda") % 3 == 0, 0.0, 1.0) if weights else None
    off = torch.arange(T, device="cuda") % 5 == 2
    p.teacher[off] = -math.inf
    p.teacher[::2, 0] = -math.inf  # and some first entries alone
    ids = p.ids.clone()
    p.ids[off] = -1
    clean = p.distill(1.5), p.distill(1.5, grads=False)["loss"]
    p.ids = ids
    check_distill(p, 1.5)
    p.H[off, 1] = math.nan
    p.H[2] = math.inf
    got = p.distill(1.5), p.distill(1.5, grads=False)["loss"]
    for key in clean[0]:
        assert bool(torch.isfinite(clean[0][key]).all()), key
        assert torch.equal(got[0][key], clean[0][key]), key
    assert torch.equal(got[1], clean[1]) and bool((got[1][off] == 0).all())
    # an id past the vocabulary is reported whatever its logit
    p.ids[2, 3] = V
    if weights:
        p.weight[2] = 1
    assert math.isnan(float(p.distill(1.5)["loss"][2]))


@gpu
def test_a_step_counts_no_row_of_minus_infinity():
    """The trainer's mean is over rows with an entry."""
    import numpy as np

    import lora_ce
    T, V, d, r, K = 40, 500, 64, 4, 3
    rng = np.random.default_rng(5)
    W = (rng.standard_normal((V, d)) / 8).astype(np.float16)
    H = rng.standard_normal((T, d)).astype(np.float32)
    ids = rng.integers(0, V, (T, K)).astype(np.int32)
    z = rng.standard_normal((T, K)).astype(np.float32)
    losses = []
    for absent in (True, False):
        m = lora_ce.LoraCE(lora_ce.default_config(d, V, r, T))
        m.set_weight(W.view(np.uint16))
        m.set_adapter(np.full((d, r), 0.1, np.float32),
                      np.full((r, V), 0.01, np.float32), 0)
        i, t, h = ids.copy(), z.copy(), H.copy()
        if absent:
            i[5:20] = -1
        else:
            t[5:20] = -np.inf
            h[5:20, 3] = np.nan
        losses.append(m.distill_step(h, i, t, 1.0))
        losses.append(m.get_adapter()[1].copy())
        m.close()
    assert losses[0] == losses[2] and np.isfinite(losses[0])
    assert np.isfinite(losses[1]).all() and np.array_equal(losses[1], losses[3])


def _same_bits(a, b):
    import torch
    return all(torch.equal(a[key], b[key]) for key in a)


@gpu
@pytest.mark.parametrize("e", [-24, -18, 18, 24])
@pytest.mark.parametrize("T,V,d,r,k", [(9, 49152, 64, 4, 8), (25, 49152, 64, 4, 8), (300, 4099, 640, 3, 8),
                                       (40, 3000, 576, 1, 60), (1300, 1000, 64, 2, 0)])
def test_low_ranks_have_the_range_of_f32(T, V, d, r, k, e):
    """A power of two moved from B to A changes no bit of what ranks up to 4 compute,
    far past f16's range, in any path: the products are the same f32 products."""
    p = Problem(T, V, d, r)
    p.lists(8)
    score, full, loss = p.score(k), p.distill(1.5), p.distill(1.5, grads=False)
    p.A *= 2.0**e
    p.B *= 2.0**-e
    assert _same_bits(p.score(k), score)
    assert p.torch.equal(p.distill(1.5, grads=False)["loss"], loss["loss"])
    got = p.distill(1.5)
    got["gA"] *= 2.0**e
    got["gB"] *= 2.0**-e
    assert _same_bits(got, full)
    check_score(p, k, p.score(k))
    check_distill(p, 1.5)


class Pairs(Problem):
    """The rank term of f16 pairs: hi + lo is off by at most 2^-25 (the spacing of
    subnormal f16 is 2^-24) or 2^-23 of the value, lo . lo is left out, 2^-22 of a
    product at most.  So each of r products is off by 2^-25 (|s U| + |B|) + 2^-21 |s U| |B|."""

    def tol(self):
        u = float((self.scale * (self.H.half().float() @ self.A)).abs().max())
        b = float(self.B.abs().max())
        return super().tol() + self.r * (2.0**-25 * (u + b) + 2.0**-21 * u * b)


@gpu
@pytest.mark.parametrize("r", [8, 16, 33])
@pytest.mark.parametrize("T", [40, 300])
def test_operands_past_f16_are_infinite_at_higher_ranks(T, r):
    """From rank 5 on the rank term's operands are pairs of f16: up to 65,504 they are
    read, past it a position's s U makes its own results NaN."""
    import torch
    p = Pairs(T, 1000, 64, r, "f32")
    p.B /= 32.0
    p.A *= 32.0
    p.H[7] *= 4096.0  # s U of about 2^18
    p.lists(8)
    out, d = p.score(5), p.distill(1.0, grads=False)["loss"]
    assert math.isnan(float(out["logprob"][7])) and bool((out["ids"][7] == -1).all())
    assert math.isnan(float(d[7])) and bool(p.distill(1.0)["gB"].isnan().all())
    rest = torch.arange(T, device="cuda") != 7
    p.H[7] = p.H[6]
    want = p.score(5)
    for key in out:
        assert torch.equal(out[key][rest], want[key][rest]), key
    check_score(p, 5, want)
    check_distill(p, 1.0)


class Cancelling(Problem):
    """Two channels of the hidden state far above the others whose parts of every
    logit cancel, the first and the last of the sum (or, in the adapter, of h . A):
    partial sums up to 100 times the logits."""

    def __init__(self, T, V, d, r, adapter=False, by=512.0):
        super().__init__(T, V, d, r)
        torch = self.torch
        a = (0.5 + self.u(V)).half()
        self.W[:, 0] = self.W[:, d - 1] = 0 if adapter else a
        if r:
            b = 0.5 + self.u(r)
            self.A[0] = self.A[d - 1] = b if adapter else 0
        K = by * 2.0 ** torch.arange(T, device="cuda").remainder(3).neg()
        self.H[:, 0], self.H[:, d - 1] = K.to(self.H.dtype), -K.to(self.H.dtype)


@gpu
@pytest.mark.parametrize("T,V,d,r,k,adapter", [
    (9, 49152, 576, 0, 64, False), (24, 49152, 576, 16, 64, True),
    (100, 49152, 576, 0, 64, False), (300, 49152, 576, 4, 64, False), (300, 49152, 576, 64, 64, True),
    (2500, 49152, 576, 0, 64, False), (200, 4099, 640, 8, 20, True), (60, 140000, 128, 33, 100, False),
    (500, 1000, 320, 3, 100, True),
])
def test_order_of_logits_whose_sums_cancel(T, V, d, r, k, adapter):
    """Ids are those of the 64-bit logits where an f32 sum's rounding, which follows
    its partial sums, is far above what the logits' own size suggests."""
    p = Cancelling(T, V, d, r, adapter)
    check_score(p, k, p.score(k))


@gpu
@pytest.mark.parametrize("r", [4, 8, 16, 64])
@pytest.mark.parametrize("T", [12, 100, 300])
@pytest.mark.parametrize("e", [-118, -60, 0])
def test_gradients_of_a_tiny_adapter(T, r, e):
    """The scale that brings B into f16's range is itself past f32's where B is tiny."""
    p = Problem(T, 1000, 64, r)
    p.lists(8)
    p.B *= 2.0**e
    check_distill(p, 1.0)


@gpu
@pytest.mark.parametrize("T,r", [(16, 0), (17, 4), (23, 16), (24, 0), (24, 4), (24, 9), (25, 0), (25, 4),
                                 (25, 16), (8, 33), (16, 33), (17, 33), (16, 64), (17, 64)])
@pytest.mark.parametrize("V,d,k", [(20001, 128, 8), (49152, 576, 20), (2048, 640, 5)])
def test_score_on_both_sides_of_few_positions(T, r, V, d, k):
    """Up to 24 positions (16 above rank 16) have a pass of their own where records
    have 64 columns, as they do here."""
    p = Problem(T, V, d, r)
    check_score(p, k, p.score(k))


@gpu
@pytest.mark.parametrize("T,r", [(16, 4), (17, 4), (31, 8), (32, 1), (32, 16), (33, 4), (33, 8), (33, 16),
                                 (16, 33), (17, 33), (16, 64), (17, 64)])
@pytest.mark.parametrize("V,d,K", [(4099, 128, 8), (20001, 576, 33)])
@pytest.mark.parametrize("grads", [True, False])
def test_distill_on_both_sides_of_few_positions(T, r, V, d, K, grads):
    """The same limit is 32 positions, 16 above rank 16."""
    p = Problem(T, V, d, r)
    p.lists(K)
    check_distill(p, 1.5, grads)


def check_elements(p, tau):
    """Every element of gA and gB by itself, against the sum of its absolute terms N.
      * a probability, and with it a term, is off by tol of itself (test_head.py)
      * the sums of the terms: 64 accumulations in f32 at a time, 2^-17 of N, and the
        f16 pairs of their operands, 2^-21; 2^-16 for both
      * s U in f32, a sum in eight parts of d / 8: d / 8 + 8 roundings of the sum of its
        absolute terms, which stands for |U| in gB's N
      * gB's sparse part is in units of 2^-38 of the largest |w s U| tau at least, and
        its operand is a pair of f16 in units of 2^-39 of it: 2^-37 per position"""
    import torch
    out = p.distill(tau)
    _, gA, gB, _, _ = p.distill64(tau)
    w = torch.ones(p.T, dtype=torch.float64, device="cuda") if p.weight is None else p.weight.double()
    ids = p.ids.long()
    t = torch.where(ids >= 0, p.teacher.double() / tau, -math.inf)
    counted = (t > -math.inf).any(1) & (w != 0)
    q = torch.softmax(torch.where(counted[:, None], t, 0.0), 1) * ((ids >= 0) & counted[:, None])
    H = p.H.half().double()
    A, B, s = p.A.double(), p.B.double(), abs(p.scale)
    dz = torch.softmax((H @ p.W.double().T + p.scale * (H @ A) @ B) / tau, 1)
    dz = dz.scatter_add_(1, ids.clamp(min=0), q) * (w.abs() * counted * tau)[:, None]
    U, U_abs = (H @ A).abs(), H.abs() @ A.abs()
    rel = p.tol() / tau + 2.0**-20 + 2.0**-16
    NA = s * (H.abs().T @ (dz @ B.abs().T))
    bound = rel * s * (U.T @ dz) + (p.d / 8 + 8) * 2.0**-24 * s * (U_abs.T @ dz)
    bound = bound + p.T * 2.0**-37 * s * float((U * (w.abs() * tau)[:, None]).max())
    assert bool(((out["gA"].double() - gA).abs() <= rel * NA + 1e-44).all())
    assert bool(((out["gB"].double() - gB).abs() <= bound).all())


@gpu
@pytest.mark.parametrize("T,V,d,r,K,tau,dtype", [
    (5, 20001, 576, 4, 8, 1.0, "bf16"), (32, 1000, 64, 16, 20, 2.0, "f16"), (16, 4099, 128, 64, 64, 1.0, "bf16"),
    (100, 4099, 576, 3, 33, 1.0, "f32"), (255, 4099, 128, 8, 20, 2.0, "bf16"),
    (300, 4099, 128, 16, 33, 1.0, "bf16"), (700, 3000, 192, 64, 10, 1.5, "bf16"),
    (2000, 1000, 64, 32, 8, 0.5, "f16"), (129, 49152, 576, 33, 64, 1.0, "bf16"),
    (4000, 777, 64, 4, 128, 4.0, "bf16"),
])
@pytest.mark.parametrize("weights", [None, "uniform", "masked"])
def test_every_element_of_the_gradients(T, V, d, r, K, tau, dtype, weights):
    p = Problem(T, V, d, r, dtype)
    p.lists(K)
    if weights:
        p.weight = p.u(T) * (p.u(T) < (0.4 if weights == "masked" else 2.0))
    check_elements(p, tau)


@gpu
@pytest.mark.parametrize("r", [4, 16])
def test_a_distillation_step_through_a_communicator(r):
    """A communicator of one rank: the sums go through its all-reduce and come back the
    same bits."""
    import numpy as np

    import lora_ce
    T, V, d, K = 60, 700, 128, 4
    rng = np.random.default_rng(r)
    W = (rng.standard_normal((V, d)) / 8).astype(np.float16)
    A, B = rng.standard_normal((d, r)).astype(np.float32) / 8, rng.standard_normal((r, V)).astype(np.float32) / 20
    H = rng.standard_normal((T, d)).astype(np.float32)
    ids, z = rng.integers(-1, V, (T, K)).astype(np.int32), rng.standard_normal((T, K)).astype(np.float32)
    weight = (rng.random(T) < 0.7).astype(np.float32)
    got = []
    for comm in (False, True):
        m = lora_ce.LoraCE(lora_ce.default_config(d, V, r, T, clip_norm=0.5))
        m.set_weight(W.view(np.uint16))
        m.set_adapter(A, B, 0)
        if comm:
            m.comm_init(1, 0, lora_ce.LoraCE.nccl_unique_id())
        got.append([m.distill_step(H, ids, z, 2.0, weight) for _ in range(2)] + list(m.get_adapter()) +
                   list(m.get_grads()))
        m.close()
    for a, b in zip(*got):
        assert np.array_equal(a, b)
    assert got[0][4] == 2
