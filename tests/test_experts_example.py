"""examples/cluster_experts.py: fitted centers, routing, grouping, products, combination and their gradients together."""
import importlib.util
import os

import pytest

from conftest import ROOT


@pytest.mark.gpu
def test_cluster_experts_learn_what_one_map_cannot(cuda_device):
    spec = importlib.util.spec_from_file_location("cluster_experts", os.path.join(ROOT, "examples", "cluster_experts.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    single, final = mod.main(rows=4000, steps=120, quiet=True)
    assert final < 0.2 * single
