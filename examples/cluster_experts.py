"""Clusters as experts: fit, route, train, compress to 4 bits, serve.

    python examples/cluster_experts.py [--rows N] [--clusters E] [--steps S]

k-means finds clusters of the tokens; every token goes to the linear models of its two nearest
centres, whose results are joined by a softmax over the distances. The models learn by gradient
descent through combine, product and dispatch. Then each is compressed to 4-bit codes of a codebook
that k-means finds for its values, and single tokens are served from those; and to microscaled 4-bit
numbers, which are multiplied with tokens in such numbers.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from h2o4gpu_amd import KMeans, codebook4, experts, microscale4  # noqa: E402


def forward(x, distances, W, top_k, scale):
    chosen, weights = experts.route(distances, top_k, largest=False, scale=scale)
    order = experts.sort_by_expert(chosen, W.shape[0])
    rows = experts.product(experts.dispatch(x, order), W, order)
    return experts.combine(rows, weights, order)


def serve(x, distances, packed, top_k, scale):
    """The same with 4-bit models: a codebook's, or microscaled ones and the tokens in 4 bits too."""
    chosen, weights = experts.route(distances, top_k, largest=False, scale=scale)
    order = experts.sort_by_expert(chosen, packed.n_experts)
    if isinstance(packed, microscale4.Microscale4):
        rows = microscale4.experts_product(microscale4.quantize(x), packed, order)
    else:
        rows = codebook4.experts_product(x, packed, order)
    return experts.combine(rows, weights, order)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--rows", type=int, default=20_000)
    ap.add_argument("--cols", type=int, default=64)
    ap.add_argument("--out", type=int, default=48)
    ap.add_argument("--clusters", type=int, default=16)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--top-k", type=int, default=2)
    ap.add_argument("--quiet", action="store_true")
    a = ap.parse_args(argv)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(7)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    # tokens of several kinds, each kind with a linear map of its own
    centres = 3 * randn(a.clusters, a.cols)
    kind = torch.randint(0, a.clusters, (a.rows,), device="cuda", generator=gen)
    x = centres[kind] + randn(a.rows, a.cols)
    maps = randn(a.clusters, a.out, a.cols) / a.cols ** 0.5
    y = (maps[kind] @ x[:, :, None])[:, :, 0]

    model = KMeans(n_clusters=a.clusters, init="k-means++", max_iter=20, random_state=3).fit(x)
    distances = model.transform(x)
    scale = 1.0 / a.cols

    W = (0.02 * randn(a.clusters, a.out, a.cols)).requires_grad_()
    adam = torch.optim.Adam([W], lr=0.02)
    losses = []
    for step in range(a.steps):
        loss = (forward(x, distances, W, a.top_k, scale) - y).square().mean()
        adam.zero_grad()
        loss.backward()
        adam.step()
        losses.append(float(loss.detach()))
        if not a.quiet and step % 10 == 0:
            print("step %d: loss %.4f" % (step, losses[-1]))

    packed = codebook4.quantize(W.detach(), group=32)
    with torch.no_grad():
        full = forward(x, distances, W, a.top_k, scale)
        small = serve(x, distances, packed, a.top_k, scale)
        error = float((small - full).norm() / full.norm())
        one = serve(x[:1], distances[:1], packed, a.top_k, scale)
        same = float((one - small[:1]).abs().max() / small[:1].abs().max())
        four = serve(x, distances, microscale4.quantize(W.detach()), a.top_k, scale)
        four_error = float((four - full).norm() / full.norm())
    if not a.quiet:
        print("loss %.4f -> %.4f; served with 4 bits: %.2f%% from the trained models, %.2f%% with the tokens in 4 bits"
              % (losses[0], losses[-1], 100 * error, 100 * four_error))
    return dict(loss_first=losses[0], loss_last=losses[-1], served_error=error, single_token=same,
                served_four_error=four_error)


if __name__ == "__main__":
    main()
