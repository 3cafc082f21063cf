"""A small model trained on 4-bit matrices: a dense layer, a router and a layer
of experts, forward and backward, every product in MX4.

    python examples/mx4_experts.py [steps]

    h = relu(x W1^T)            bsq_mx4_linear, which keeps x^T at 4.25 bits a value
    ids, p = route(h R^T)       bsq_moe_route (softmax, two of eight experts)
    y = sum of p_j h W_e^T      bsq_moe_linear
    loss = mean (y - target)^2

The weights are FP32 on the host, stepped by plain gradient descent and encoded
anew, rows and columns in one pass, before each step.  The targets come from a
model of the same shape.  Prints the loss; exits with an error if it does not
fall.
"""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bitsqueeze-llm_amd"))
import bitsqz_amd as B  # noqa: E402

TOKENS, INPUTS, HIDDEN, OUTPUTS, EXPERTS, CHOSEN = 512, 192, 256, 96, 8, 2


def weights(rng):
    return {"w1": rng.standard_normal((HIDDEN, INPUTS)).astype(np.float32) / np.sqrt(INPUTS),
            "router": rng.standard_normal((EXPERTS, HIDDEN)).astype(np.float32) * 2.0 / np.sqrt(HIDDEN),
            "w2": rng.standard_normal((EXPERTS, OUTPUTS, HIDDEN)).astype(np.float32) / np.sqrt(HIDDEN)}


def exact(p, x):
    """The model in FP32, for the targets."""
    h = np.maximum(x @ p["w1"].T, 0.0)
    logits = h @ p["router"].T
    ids = np.argsort(-logits, 1, kind="stable")[:, :CHOSEN]
    s = np.exp(np.take_along_axis(logits, ids, 1) - logits.max(1, keepdims=True))
    s /= s.sum(1, keepdims=True)
    return sum(s[:, j, None] * np.einsum("th,toh->to", h, p["w2"][ids[:, j]]) for j in range(CHOSEN))


def step(p, x, target, rate):
    """One step of gradient descent; returns the loss before it."""
    w1, w1_columns = B.mx4_encode(p["w1"], columns=True)
    router, router_columns = B.mx4_encode(p["router"], columns=True)
    experts = B.MoeLinear(*B.mx4_encode(p["w2"], columns=True))

    a, x_kept = B.mx4_linear(x, w1, keep=True)
    h = np.maximum(a, 0.0)
    logits, h_kept = B.mx4_linear(h, router, keep=True)
    ids, share = B.moe_route(logits, CHOSEN)
    y = experts.forward(h, ids, share)

    d_y = 2.0 * (y - target) / y.shape[1]  # a token's mean; averaged over tokens by `rate`
    d_h, d_share, d_w2 = experts.backward(d_y)
    d_logits = B.moe_route_backward(logits, ids, d_share)
    d_h_router, d_router = B.mx4_linear_backward(d_logits, h_kept, router_columns)
    _, d_w1 = B.mx4_linear_backward((d_h + d_h_router) * (a > 0.0), x_kept, w1_columns)
    for name, g in (("w1", d_w1), ("router", d_router), ("w2", d_w2)):
        p[name] -= rate * g
    return float(((y - target) ** 2).mean())


def train(steps=40, seed=0, rate=0.005):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((TOKENS, INPUTS)).astype(np.float32)
    target = exact(weights(rng), x).astype(np.float32)
    p = weights(rng)
    return [step(p, x, target, rate) for _ in range(steps)]


if __name__ == "__main__":
    losses = train(int(sys.argv[1]) if len(sys.argv) > 1 else 40)
    for i, v in enumerate(losses):
        if i % 5 == 0 or i + 1 == len(losses):
            print(f"step {i:3d}  loss {v:.4f}")
    sys.exit(0 if losses[-1] < losses[0] else "the loss did not fall")
