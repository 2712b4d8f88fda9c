"""Models and layers beside the options that deep stacks have: modules saved before there were any, configurations and
model classes that do not know them, and what their refusals say.  On the CPU."""
import copy
import types

import pytest
import torch

import cxgnncomp


def _as_saved_before(module):
    """The module as one restored from a file that was written before it had the options."""
    old = copy.deepcopy(module)
    for m in old.modules():
        for name in ("checkpoint", "residual"):
            m.__dict__.pop(name, None)
    return old


@pytest.mark.parametrize("kind", ["SAGE", "GCN", "GIN", "GAT", "RGCN"])
def test_modules_saved_before_the_options(kind, monkeypatch):
    more = {"GAT": dict(heads=1), "RGCN": dict(num_rel=2)}.get(kind, {})
    model = _as_saved_before(getattr(cxgnncomp, kind)(4, 8, 3, 2, 0.0, "CSR_Layer", **more))
    assert model.residual is None and model.checkpoint is None
    model.reset_parameters()
    if kind in ("SAGE", "GCN", "GIN"):
        assert all(conv.checkpoint is None for conv in model.convs)
    # the forward pass up to the layers, which need a GPU
    monkeypatch.setattr(type(model), "layer", lambda self, conv, x, batch, i: x @ torch.ones(x.shape[1], 8 if i == 0 else 3))
    batch = types.SimpleNamespace(x=torch.randn(5, 4), ptr=torch.zeros(6, dtype=torch.long), idx=torch.zeros(0, dtype=torch.long),
                                  etypes=torch.zeros(0, dtype=torch.long))
    assert tuple(model(batch).shape) == (5, 3)


def _config(**model):
    ns = types.SimpleNamespace
    return ns(dl=ns(dataset=ns(feature_dim=8, num_classes=4, name="x"), sampler=ns(train=ns(num_layer=3))),
              train=ns(type="cxg", model=dict(hidden_dim=16, dropout=0.0, **model)))


def test_configurations_without_the_options(monkeypatch):
    """A model class of the user's own in model_dict that takes neither option, and options that are off."""

    class Mine(torch.nn.Module):
        def __init__(self, infeat, hidden, outfeat, num_layer, dropout, graph_type, config=None):
            super().__init__()
            self.args = (infeat, hidden, outfeat, num_layer, dropout, graph_type)

    monkeypatch.setitem(cxgnncomp.model_dict, "mine", Mine)
    assert cxgnncomp.get_model(_config(type="mine")).args == (8, 16, 4, 3, 0.0, "CSR_Layer")
    with pytest.raises(TypeError):
        cxgnncomp.get_model(_config(type="mine", residual="rms"))
    for off in (None, False):
        m = cxgnncomp.get_model(_config(type="gcn", residual=off, checkpoint=off))
        assert m.residual is None and m.checkpoint is None and len(m.bns) == 2
    m = cxgnncomp.get_model(_config(type="gcn", residual="layer", checkpoint="e4m3"))
    assert m.residual == "layer" and m.checkpoint == "e4m3"
    with pytest.raises(ValueError):
        cxgnncomp.get_model(_config(type="gcn", residual="batch"))


@pytest.mark.parametrize("kind,more", [("GAT", dict(heads=1)), ("RGCN", dict(num_rel=2))])
def test_models_that_do_not_take_a_checkpoint_say_who_does(kind, more):
    """(They do keep inputs of linear maps, in fp32: the refusal must not say otherwise.)"""
    with pytest.raises(ValueError, match="taken by SAGE, GCN and GIN") as refusal:
        getattr(cxgnncomp, kind)(4, 8, 3, 2, 0.0, "CSR_Layer", checkpoint="int8", **more)
    assert kind in str(refusal.value)
