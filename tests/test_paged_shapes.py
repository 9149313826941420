"""Shapes that the Python mirror of the paged cache takes: right ones in more than one form, and none whose elements only happen
to be as many."""
import pytest
import torch

from tests.test_paged_refusals import _args, kv  # noqa: F401

BF = torch.bfloat16


def _t(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


# the layer: 3 tokens, 4 query heads, 2 key heads, head_dim 64, 16 pairs turned
@pytest.mark.parametrize("name,tensor", [("Q", _t(4, 3, 64)), ("Q", _t(3, 64, 4)), ("K", _t(2, 3, 64)), ("V", _t(64, 3, 2)), ("V", _t(2, 192)),
                                         ("Q_out", _t(4, 3, 64)), ("Q_out", _t(3 * 4 * 64)), ("K", _t(6, 64)), ("K", _t(3, 64, 2))])
def test_tensors_in_another_order_are_refused(kv, name, tensor):  # noqa: F811
    from f2k_cuda_b200 import paged
    with pytest.raises(TypeError):
        kv.append(**{**_args(), name: tensor})
    assert not paged.lib.calls


def test_tables_and_lse_in_another_order_are_refused(kv):  # noqa: F811
    from f2k_cuda_b200 import paged
    a = _args()
    turned = _t(16, 40, dtype=torch.float32)
    for tables in ((turned, turned), (a["tables"][0], turned)):
        with pytest.raises(TypeError):
            kv.append(**{**a, "tables": tables})
    with pytest.raises(TypeError):
        kv.attend(a["Q"], a["Q_out"], a["batch"], None, lse=_t(4, 3, dtype=torch.float32))
    assert not paged.lib.calls


def test_other_forms_of_the_same_layout_are_taken(kv):  # noqa: F811
    from f2k_cuda_b200 import paged
    a = _args()
    assert kv.append(**{**a, "Q": _t(3, 256), "K": _t(3, 128), "V": _t(1, 3, 2, 64), "Q_out": _t(3, 1, 4, 64)})
    assert kv.attend(_t(3, 1, 4, 64), _t(3, 256), a["batch"], None, lse=_t(3, 4, dtype=torch.float32))
    assert kv.attend(a["Q"], a["Q_out"], a["batch"], None, lse=_t(12, dtype=torch.float32))
    assert len(paged.lib.calls) == 3
