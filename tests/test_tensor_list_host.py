"""TensorList beside the arguments that it replaces: refused, not dropped."""
import pytest
import torch

import coconet_b200 as coco

HYPER = (1e-3, 0.9, 0.999, 1e-8, 0.0, 0)


def _call(comm, quant, lst, ws=None, **kw):
    t = torch.zeros(256)
    if quant:
        st = coco.quant_state([256], 1, device="cpu")
        comm.fused_adamw_quant_scattered(lst, ws, *st, *HYPER, 0, **kw)
    else:
        comm.fused_adamw_scattered(lst, ws, t, t.clone(), *HYPER, **kw)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("what", ["ws", "w_lps", "no_decay"])
def test_arguments_beside_a_tensor_list_are_refused(quant, what):
    comm = coco.Communicator(None, 1, 0)   # never reaches the library
    g, w = torch.zeros(256), torch.zeros(256)
    lst = coco.TensorList([g], [w])
    other = {"ws": [w.clone()], "w_lps": [w.bfloat16()], "no_decay": [True]}[what]
    with pytest.raises(ValueError, match=f"TensorList.*{what}"):
        _call(comm, quant, lst, **{what: other})
    full = coco.TensorList([g], [w], lps=[w.half()], no_decay=[False])
    with pytest.raises(ValueError, match=f"TensorList.*{what}"):
        _call(comm, quant, full, **{what: other})
    with pytest.raises(ValueError, match=f"TensorList.*{what}"):
        _call(comm, quant, full, **{what: []})


@pytest.mark.parametrize("quant", [False, True])
def test_a_tensor_list_by_itself_goes_on_to_the_other_checks(quant):
    comm = coco.Communicator(None, 1, 0)
    lst = coco.TensorList([torch.zeros(256)], [torch.zeros(256)], no_decay=[True])
    with pytest.raises(ValueError, match="CUDA"):
        _call(comm, quant, lst)
    g, w, lp = torch.zeros(256), torch.zeros(256), torch.zeros(256).half()
    lst = coco.TensorList([g], [w], lps=[lp], no_decay=[True])
    with pytest.raises(ValueError, match="CUDA"):   # the same once more is no contradiction
        _call(comm, quant, lst, ws=[w], w_lps=[lp], no_decay=[1])
    with pytest.raises(ValueError, match="CUDA"):   # and plain lists keep their arguments
        _call(comm, quant, [torch.zeros(256)], [torch.zeros(256)], no_decay=[True], w_lps=[torch.zeros(256).half()])
