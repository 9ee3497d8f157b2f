"""What the calls of the coded cache refuse on the host.  No GPU."""
import pytest
import torch

from glint_b200 import ops_cache8
from glint_b200.errors import KernelError
from tests.test_cache8 import _pretend, _step

i32 = lambda *v: torch.tensor(v, dtype=torch.int32)


def _mixed(contexts, lens, max_context=100):
    T, R = sum(lens), len(lens)
    return _step(T, pages=8, seq_start=torch.zeros(R, dtype=torch.int32), cu_seqlens=torch.zeros(R + 1, dtype=torch.int32),
                 block_table=torch.zeros(R, 8, dtype=torch.int32), max_seq_len=max(lens), max_context=max_context, contexts=contexts)


@pytest.mark.parametrize("contexts,lens", [([5, 9, 3], [1, 1, 0]),          # more single tokens than there are tokens
                                           ([5, 9], [1, 3]),                # a request of three among them
                                           ([5, 9], [0, 2]), ([5, 9], [2, 0, 0]),
                                           ([0], [1, 3]), ([-3], [1]), ([101], [1, 3])])
def test_contexts_that_do_not_fit_the_step(monkeypatch, contexts, lens):
    """The launches take the requests in front as a token each: more of them than tokens, or none behind with the rest, would be
    read past the arrays' end or left out."""
    _pretend(monkeypatch)
    with pytest.raises(KernelError, match="context"):
        _mixed(contexts, lens)


@pytest.mark.parametrize("contexts,lens", [([], [1, 3]), ([7], [1, 3]), ([7, 100], [1, 1]), ([7], [1, 0, 1]), ([7], [1, 1, 40]), ([], [0, 0])])
def test_contexts_that_do(monkeypatch, contexts, lens):
    _pretend(monkeypatch)
    assert _mixed(contexts, lens).struct.leading_single == (len(lens) if max(lens) == 1 else len(contexts))


@pytest.mark.parametrize("missing", [("v_pool",), ("k_scale",), ("v_scale",), ("k_pool", "v_pool"), ("status",)])
def test_an_operand_left_out_is_refused(monkeypatch, missing):
    _pretend(monkeypatch)
    z = lambda *shape, dtype=torch.float32: torch.zeros(*shape, dtype=dtype)
    args = dict(qkv=z(3, 8 * 32), positions=i32(0, 1, 2), token_seq=i32(0, 0, 0), block_table=z(1, 3, dtype=torch.int32), turns=z(16, dtype=torch.float64),
                q_out=z(3, 4 * 32), k_pool=z(3, 2, 16, 32, dtype=torch.uint8), v_pool=z(3, 2, 16, 32, dtype=torch.uint8),
                nh=4, nkv=2, hd=32, page_size=16, num_pages=3, status=i32(0), k_scale=z(3, 2), v_scale=z(3, 2))
    args.update({name: None for name in missing})
    with pytest.raises(KernelError, match="pool|scale|status"):
        ops_cache8.ops.rope_append(**args)
