"""Layers built from a configuration record that has the reference's fields and nothing else (its own
LayerCfg, a namespace): what is beside them is off."""
import dataclasses
from types import SimpleNamespace

import pytest
import torch

from sca2_b200 import layers


def _record(**kw):
    cfg = layers.LayerCfg(d=32, Mc=16, Md=4, G=4, ff=48, freq="rope", dv=32, **kw)
    return cfg, SimpleNamespace(**{f.name: getattr(cfg, f.name) for f in dataclasses.fields(cfg) if f.name != "tail"})


@pytest.mark.parametrize("cls", ["SCA2Layer", "GatedLayer", "ShortLayer", "ShortLayerDampH"])
def test_record_without_a_tail(cls):
    cfg, ref = _record()
    built = []
    for c in (cfg, ref):
        torch.manual_seed(3)
        built.append(getattr(layers, cls)(c).state_dict())
    assert built[0].keys() == built[1].keys()
    assert all(torch.equal(built[0][k], built[1][k]) for k in built[0])
