"""Positions that a caller's block table has no room for, through every kernel that attention over coded pages may take: reported,
never read past the table, never a walk of its own length; other requests are what they are without them."""
import pytest
import torch

from tests.test_cache8_gpu import DEV, Setup, rts  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,lens,starts,nh,nkv,hd,P", [
    ("float32", [1, 1, 1], [3, 40, 20], 2, 1, 32, 16),            # the kernel of the 32-bit path
    ("float32", [5, 30, 7], [3, 40, 20], 2, 1, 36, 12),
    ("bfloat16", [5, 30, 7], [3, 40, 20], 4, 2, 64, 16),          # portions
    ("bfloat16", [5, 300, 7], [300, 700, 20], 4, 2, 128, 16),     # portions whose keys are split
    ("bfloat16", [5, 30, 7], [3, 40, 20], 4, 2, 64, 48),          # prompts over other pages
    ("bfloat16", [5, 30, 7], [3, 40, 20], 71, 1, 64, 128),        # many query heads a kv head
    ("bfloat16", [5, 30, 7], [3, 40, 20], 4, 2, 36, 12),          # head sizes that no tensor-core kernel takes
])
@pytest.mark.parametrize("window", [0, 20])
def test_positions_outside_the_block_table(rts, dtype, lens, starts, nh, nkv, hd, P, window):
    from glint_b200 import ops_cache8
    from glint_b200.errors import KernelError
    rt = rts[dtype]
    s = Setup(rt, lens, starts, nkv, hd, P, seed=3)
    T = sum(lens)
    q = (0.1 * torch.randn(T, nh * hd, generator=torch.Generator().manual_seed(1))).to(DEV, rt.dtype)
    good = ops_cache8.attention(rt, s.cache, s.step, q, nh, 1.0, window=window)
    rt.check_status()
    others = torch.ones(T, dtype=torch.bool, device=DEV)
    others[lens[0]:lens[0] + lens[1]] = False
    room = s.table.shape[1] * P
    for far in (room - lens[1] + 1, room, room + 1000, 2 ** 31 - 1 - lens[1]):
        s.step.tensors["positions"][lens[0]:lens[0] + lens[1]] = far + torch.arange(lens[1], dtype=torch.int32, device=DEV)
        s.step.tensors["seq_start"][1] = far
        s.step.begin()
        out = ops_cache8.attention(rt, s.cache, s.step, q, nh, 1.0, window=window)
        with pytest.raises(KernelError, match="attention read"):
            rt.check_status()
        assert torch.equal(out[others], good[others]), far
