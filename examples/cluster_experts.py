"""A mixture of linear experts on fitted centers: KMeans finds the clusters, a row goes to the experts of its two
nearest centers, and the experts' matrices and the router's centers are trained together.

    python examples/cluster_experts.py [--rows 20000] [--dims 24] [--clusters 8] [--steps 200]

Every cluster of the synthetic data has a linear law of its own, which one linear map cannot follow.  The steps are the
library's: KMeans.fit, then per training step route -> group_rows -> expert_matmul -> combine_rows and their gradients.
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from mlx_kmeans_b200 import KMeans, combine_rows, expert_matmul, group_rows, make_data_numpy, route  # noqa: E402


class ClusterExperts(torch.nn.Module):
    """out_t = sum over the top_k nearest centers c_e of p_e W_e [x_t, 1], p the softmax of -|x_t - c_e|^2 / tau."""

    def __init__(self, centers, outputs, top_k=2, tau=1.0):
        super().__init__()
        k, d = centers.shape
        self.centers = torch.nn.Parameter(centers.clone())
        self.weight = torch.nn.Parameter(torch.zeros(k, outputs, d + 1, device=centers.device))
        self.top_k, self.tau = top_k, tau

    def logits(self, x):
        # -|x - c|^2 / tau without its |x|^2, which the softmax does not see
        return (2.0 * x @ self.centers.T - self.centers.square().sum(1)) / self.tau

    def forward(self, x):
        ids, weights = route(self.logits(x), self.top_k)
        groups = group_rows(ids, len(self.centers))
        ones = torch.ones(len(x), 1, device=x.device)
        y = expert_matmul(torch.cat([x, ones], 1).bfloat16(), self.weight.bfloat16(), groups)
        return combine_rows(y.float(), groups, weights)


def main(rows=20000, dims=24, clusters=8, steps=200, outputs=5, seed=0, quiet=False):
    rng = np.random.default_rng(seed)
    X = make_data_numpy(rows, dims, clusters, seed)[0]
    X = (X - X.mean(0)) / X.std()
    km = KMeans(n_clusters=clusters, random_state=seed, n_init=2).fit(X)
    laws = rng.standard_normal((clusters, outputs, dims)).astype(np.float32) / np.sqrt(dims)
    shift = rng.standard_normal((clusters, outputs)).astype(np.float32)
    lab = np.asarray(km.labels_)
    Y = np.einsum("tod,td->to", laws[lab], X) + shift[lab]
    x, y = torch.from_numpy(X).cuda().float(), torch.from_numpy(Y).cuda().float()

    ones = torch.ones(rows, 1, device="cuda")
    one_map = torch.linalg.lstsq(torch.cat([x, ones], 1), y).solution
    single = float((torch.cat([x, ones], 1) @ one_map - y).square().mean())

    centers = torch.as_tensor(np.asarray(km.cluster_centers_), dtype=torch.float32, device="cuda")
    model = ClusterExperts(centers, outputs, tau=0.25 * float(torch.cdist(centers, centers).square().mean()))
    opt = torch.optim.Adam([{"params": [model.weight], "lr": 0.05}, {"params": [model.centers], "lr": 0.002}])
    for step in range(steps):
        loss = (model(x) - y).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        if not quiet and step % 50 == 0:
            print(f"step {step:4d}  mean square error {loss.item():.5f}")
    with torch.no_grad():
        final = float((model(x) - y).square().mean())
    if not quiet:
        print(f"one linear map {single:.5f}, {clusters} experts on the fitted centers {final:.5f}")
    return single, final


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("rows", 20000), ("dims", 24), ("clusters", 8), ("steps", 200)):
        p.add_argument(f"--{name}", type=int, default=value)
    main(**vars(p.parse_args()))
