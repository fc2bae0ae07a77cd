"""Train a per-atom energy head on a DeepPot's descriptors.

    python examples/train_head.py [steps]

Takes a few water cells, lets a DeepPot evaluate them (descriptors and atom energies),
and trains a head on the frozen descriptors to give those energies:

    x_i = [D_i | E[t_i]]             the descriptor and a type embedding (ops.embed, into its columns)
    e_i = (silu(x_i Wg) * (x_i Wu)) Wd               the gated block (ops.gated_forward)
    loss = mean (e_i - target_i)^2

The backward gives the weights' gradients and dx, whose last columns are the gradient of
the embedded rows (ops.gated_backward, ops.embed_grad); Adam runs on the host. All
arrays of the head stay on the GPU but for the parameters' update.
"""
import importlib
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

WIDTH, HIDDEN = 16, 240  # of the type embedding and of the block


def data(dp, cells=4, seed=0):
    """Standardised descriptors, types and centred atom energies of `cells` water cells."""
    pot = dp.DeepPot(file_content=dp.model.to_bytes(dp.model.random_model("water", seed=1000)))
    d, t, e = [], [], []
    for k in range(cells):
        coord, atype, box = dp.systems.water(4, 12.42, seed=seed + k)
        energy = pot.compute(coord, atype, box, atomic=True)[3]
        d.append(pot.stage(dp.STAGE_DESCRPT, np.float64, (len(atype), pot.ndescrpt)))
        t.append(np.asarray(atype, np.int32))
        e.append(energy)
    d, t, e = np.concatenate(d), np.concatenate(t), np.concatenate(e)
    d = (d - d.mean(0)) / (d.std(0) + 1e-6)
    for k in range(pot.numb_types()):
        e[t == k] -= e[t == k].mean()
    return d.astype(np.float32), t, (e / e.std()).astype(np.float32)


class Adam:
    def __init__(self, shape, rate=3e-4):
        self.m, self.v, self.k, self.rate = np.zeros(shape, np.float32), np.zeros(shape, np.float32), 0, rate

    def step(self, p, g):
        self.k += 1
        self.m += 0.1 * (g - self.m)
        self.v += 0.01 * (g * g - self.v)
        a = self.rate * np.sqrt(1 - 0.99 ** self.k) / (1 - 0.9 ** self.k)
        return (p - a * self.m / (np.sqrt(self.v) + 1e-8)).astype(np.float32)


def train(dp, steps=60, cells=4):
    """The losses of the steps."""
    hip = importlib.import_module(dp.__name__ + ".hip")
    desc, types, target = data(dp, cells)
    n, d = desc.shape
    kinds, wide = int(types.max()) + 1, d + WIDTH
    st = dp.systems.Stream(7, 3)

    def normal(r, c, size):
        return (st.normal(r * c).reshape(r, c) * size).astype(np.float32)

    host = {"wg": normal(wide, HIDDEN, wide ** -0.5), "wu": normal(wide, HIDDEN, wide ** -0.5),
            "wd": normal(HIDDEN, 1, HIDDEN ** -0.5), "table": normal(kinds, WIDTH, 1.0)}
    par = {k: hip.DeviceArray(v) for k, v in host.items()}
    grad = {k: hip.DeviceArray(nbytes=v.nbytes) for k, v in host.items()}
    opt = {k: Adam(v.shape) for k, v in host.items()}
    x = hip.DeviceArray(np.concatenate([desc, np.zeros((n, WIDTH), np.float32)], 1))
    ids = hip.DeviceArray(types)
    y, dy, dx = (hip.DeviceArray(nbytes=4 * k) for k in (n, n, n * wide))
    ops = dp.ops.Operators()
    shape = dp.ops.GatedShape(n, wide, HIDDEN, 1, dtype="f32", act="silu")
    saved = hip.DeviceArray(nbytes=shape.saved_bytes())
    tail = 4 * d  # bytes before the embedded columns of a row
    losses = []
    for _ in range(steps):
        w = [par[k].ptr for k in ("wg", "wu", "wd")]
        ops.embed(ids.ptr, par["table"].ptr, x.ptr + tail, n, kinds, WIDTH, ld_out=wide)
        ops.gated_forward(shape, x.ptr, *w, y.ptr, saved=saved.ptr)
        err = y.to_host(np.float32, n) - target
        losses.append(float((err * err).mean()))
        dy.upload((2.0 / n * err).astype(np.float32))
        ops.gated_backward(shape, x.ptr, *w, saved.ptr, dy.ptr, dx.ptr, *(grad[k].ptr for k in ("wg", "wu", "wd")))
        ops.embed_grad(ids.ptr, dx.ptr + tail, grad["table"].ptr, n, kinds, WIDTH, ld_dout=wide)
        for k in host:
            host[k] = opt[k].step(host[k], grad[k].to_host(np.float32, host[k].shape))
            par[k].upload(host[k])
    return losses


if __name__ == "__main__":
    sys.path.insert(0, ROOT)
    result = train(importlib.import_module("dpa4c-scale-aware-md_amd"), int(sys.argv[1]) if len(sys.argv) > 1 else 60)
    for step in range(0, len(result), max(1, len(result) // 10)):
        print(f"step {step:4d}  loss {result[step]:.4f}")
    print(f"step {len(result) - 1:4d}  loss {result[-1]:.4f}")
