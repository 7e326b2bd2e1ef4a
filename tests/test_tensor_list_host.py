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


@pytest.mark.parametrize("what", ["weight", "copy"])
def test_a_tensor_that_is_written_twice_is_refused(what):
    comm = coco.Communicator(None, 1, 0)
    g, w, lp = ([torch.zeros(64) for _ in range(2)] for _ in range(3))
    lp = [x.half() for x in lp]
    if what == "weight":
        w[1] = w[0]
    else:
        lp[1] = lp[0].view(8, 8)
    with pytest.raises(ValueError, match=f"{what} twice"):
        comm.fused_adamw_scattered(g, w, w[0], w[0], *HYPER, w_lps=lp)
    lst = coco.TensorList([g[0], g[0]], w, lps=lp)
    with pytest.raises(ValueError, match="CUDA"):   # the norm writes neither, and a gradient may be there twice
        comm.grad_norm_scattered(lst, torch.zeros(2))
    with pytest.raises(ValueError, match=f"{what} twice"):
        comm.fused_adamw_scattered(lst, None, w[0], w[0], *HYPER)


def test_empty_tensors_may_be_there_twice():
    e, t = torch.zeros(0), [torch.zeros(64) for _ in range(4)]
    with pytest.raises(ValueError, match="CUDA"):
        coco.Communicator(None, 1, 0).fused_adamw_scattered([t[0], e, e], [t[1], e, e], t[2], t[3], *HYPER)
