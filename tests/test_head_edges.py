"""The operators on the LoRA head (include/lora_head.h) at their edges: ties and
crowds among the alternatives, both sides of every dispatch, ranges of the operands,
sums that cancel, gradients element by element.  The tolerances are those of
test_head.py unless a test derives its own."""
import math

import pytest

from test_head import Problem, check_score

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
