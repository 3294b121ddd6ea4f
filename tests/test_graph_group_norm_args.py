"""What a captured group_norm refuses before it runs: the arguments that the eager call refuses."""
import pytest
import torch

import flagdnn_b200 as fd

X = fd.TensorSpec("x", (2, 8, 4, 4), torch.bfloat16)
W, W32, W16 = (fd.TensorSpec("w", (8,), t) for t in (torch.bfloat16, torch.float32, torch.float16))


def compiled(call, w=W):
    return fd.compile(call, inputs=[X, w], options={"cache": None})


def test_unknown_keywords():
    with pytest.raises(TypeError, match="unexpected keyword argument 'act'"):
        compiled(lambda x, w: fd.group_norm(x, 4, act="silu"))
    with pytest.raises(TypeError, match="unexpected keyword argument 'operands'"):
        compiled(lambda x, w: fd.group_norm(x, 4, operands=("weight",)))
    with pytest.raises(TypeError, match="multiple values"):
        compiled(lambda x, w: fd.group_norm(x, 4, num_groups=4))


def test_unknown_activations():
    with pytest.raises(RuntimeError, match="activation must be one of"):
        compiled(lambda x, w: fd.group_norm(x, 4, activation="tanh"))


def test_parameter_types():
    with pytest.raises(RuntimeError, match="weight must be of the input's type or float32"):
        compiled(lambda x, w: fd.group_norm(x, 4, weight=w), W16)
    with pytest.raises(RuntimeError, match="bias must be of the input's type or float32"):
        compiled(lambda x, w: fd.group_norm(x, 4, bias=w), W16)
    for w in (W, W32):
        node, = compiled(lambda x, w: fd.group_norm(x, 4, w, w, 1e-3, "gelu"), w).graph.nodes
        assert node.attrs["activation"] == "gelu" and node.attrs["operands"] == ("weight", "bias")


def test_parameters_of_two_types():
    def block(x, w, b):
        return fd.group_norm(x, 4, w, b)

    with pytest.raises(RuntimeError, match="same dtype"):
        fd.compile(block, inputs=[X, W, fd.TensorSpec("b", (8,), torch.float32)], options={"cache": None})
