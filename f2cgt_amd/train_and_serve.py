"""A GraphSAGE layer over compressed features, trained with orthogonalised updates and served with 8-bit weights:

    python -m f2cgt_amd.train_and_serve [--nodes N] [--steps K] [--seed S] [--norm] [--packed] [--learnt]

Features of a few classes are coded in 4 bits a value, a mean-aggregating layer (examples/conv.py:9-76) learns the classes
with `pipeline.Muon` on its two weights (the bias goes to SGD), `pipeline.int8_layers` codes the trained weights, and the
accuracies of both forms on blocks that were not trained on are printed.  `--norm` puts a `pipeline.LayerNorm` behind the layer,
`--packed` keeps 8-bit checkpoints for the backward pass in place of activations (`pipeline.packed_layers`), and `--learnt` adds
learnt rows (`pipeline.NodeEmbedding`) to the destination nodes' features.
"""
from __future__ import annotations

import argparse
import copy

import torch
from torch import nn

from f2cgt_amd import pipeline


def _block(nodes, rows, fanout, generator, labels):
    """(seed ids, CSC block): a row's neighbours share its class three times out of four."""
    seeds = torch.randint(0, nodes, (rows,), generator=generator, device="cuda")
    near = torch.randint(0, nodes, (rows, fanout, 4), generator=generator, device="cuda")
    same = labels[near] == labels[seeds][:, None, None]
    pick = torch.where(same.any(2), same.int().argmax(2), torch.zeros_like(near[..., 0]))
    ids = near.gather(2, pick[..., None]).flatten()
    return seeds, torch.arange(0, rows * fanout + 1, fanout, device="cuda"), ids


def run(nodes=20000, dim=100, classes=16, rows=1024, fanout=10, steps=60, seed=0, norm=False, packed=False, learnt=False):
    """-> (accuracy with fp32 weights, with 8-bit weights, share of equal answers, losses)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    torch.manual_seed(seed)
    labels = torch.randint(0, classes, (nodes,), generator=g, device="cuda")
    centres = torch.randn((classes, dim), generator=g, device="cuda")
    features = centres[labels] + 2.0 * torch.randn((nodes, dim), generator=g, device="cuda")
    table, codebooks = pipeline.sq_compress(features, 4, 104, sample_index=torch.arange(nodes))
    manager = pipeline.CompressionManager({"methods": ["sq"], "feat_dim": dim, "configs": [(104, 4)], "codebooks": [codebooks],
                                           "compression_data": table}, fusion=True)
    layer = pipeline.MySAGEConv(dim, classes, "mean", manager, norm=pipeline.LayerNorm(classes) if norm else None).cuda()
    if packed:
        pipeline.packed_layers(layer)
    rows_of = pipeline.NodeEmbedding(nodes, dim, scale=0.1).cuda() if learnt else None
    weights = [layer.fc_self.weight, layer.fc_neigh.weight]
    muon = pipeline.Muon(weights, lr=0.05, weight_decay=0.01)
    sgd = torch.optim.SGD([layer.fc_self.bias] + (list(layer.norm.parameters()) if norm else []) +
                          (list(rows_of.parameters()) if learnt else []), lr=0.05)

    def scores(of, block):
        seeds, indptr, ids = block
        h_self = manager._decompress(0, manager.data[seeds])
        if learnt:
            h_self = h_self + rows_of(seeds)
        return of((indptr, ids), (h_self, manager.data.data))

    losses = []
    for _ in range(steps):
        block = _block(nodes, rows, fanout, g, labels)
        loss = nn.functional.cross_entropy(scores(layer, block), labels[block[0]])
        muon.zero_grad()
        sgd.zero_grad()
        loss.backward()
        muon.step()
        sgd.step()
        losses.append(loss.detach())
    manager_of, layer.sm = layer.sm, None            # (the tables are shared, not copied)
    served = pipeline.int8_layers(copy.deepcopy(layer))
    layer.sm = served.sm = manager_of
    right, right8, equal, count = 0, 0, 0, 0
    with torch.no_grad():
        for _ in range(4):
            block = _block(nodes, rows, fanout, g, labels)
            full, few = scores(layer, block).argmax(1), scores(served, block).argmax(1)
            right += int((full == labels[block[0]]).sum())
            right8 += int((few == labels[block[0]]).sum())
            equal += int((full == few).sum())
            count += rows
    return right / count, right8 / count, equal / count, torch.stack(losses).cpu()


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--nodes", type=int, default=20000)
    p.add_argument("--steps", type=int, default=60)
    p.add_argument("--seed", type=int, default=0)
    p.add_argument("--norm", action="store_true")
    p.add_argument("--packed", action="store_true")
    p.add_argument("--learnt", action="store_true")
    a = p.parse_args()
    full, few, equal, losses = run(nodes=a.nodes, steps=a.steps, seed=a.seed, norm=a.norm, packed=a.packed, learnt=a.learnt)
    print("loss %.3f -> %.3f; accuracy fp32 %.3f, 8-bit weights %.3f, equal answers %.3f" %
          (losses[0], losses[-1], full, few, equal))


if __name__ == "__main__":
    main()
