"""Tokens from a small model whose weights, keys and values are all in 4 bits.

    python examples/kv4_generate.py [tokens]

Two blocks of attention and a dense layer, three requests with prompts of their
own lengths, then a token at a time for each; one request ends on the way.

    x = embedding[token]
    q, k, v = x W^T                          bsq_mx4_linear
    q, k turned, k and v into the cache      bsq_kv4_plan, bsq_kv4_append
    a = attention of q over the cache        bsq_kv4_attention
    x = x + a O^T, x = x + relu(x U^T) D^T   bsq_mx4_linear

Each layer's cache plans its own pages here; a program that calls the library
itself plans once a step, and its layers share the table and the places.

The weights are random.  At the end the tokens of the requests that go on are
computed once more, each as one prompt; prints the largest difference of the
logits of the last step, and exits with an error if it is not small: keys and values in the
cache are the same either way.
"""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bitsqueeze-llm_amd"))
import bitsqz_amd as B  # noqa: E402

VOCABULARY, LAYERS, QUERIES, HEADS, DIM, HIDDEN, PAGE = 512, 2, 8, 2, 64, 1024, 16
WIDTH = QUERIES * DIM


class Model:
    def __init__(self, seed=0):
        rng = np.random.default_rng(seed)

        def packed(n, k):
            return B.mx4_encode(rng.standard_normal((n, k)).astype(np.float32) / np.sqrt(k))

        self.embedding = rng.standard_normal((VOCABULARY, WIDTH)).astype(np.float32)
        self.layers = [{"qkv": packed((QUERIES + 2 * HEADS) * DIM, WIDTH), "o": packed(WIDTH, WIDTH),
                        "up": packed(HIDDEN, WIDTH), "down": packed(WIDTH, HIDDEN)} for _ in range(LAYERS)]
        self.head = packed(VOCABULARY, WIDTH)
        self.turn = B.Turn(*B.rope_frequencies(DIM, 10000.0, B.ROPE_PARTS, 4.0, 64.0))

    def caches(self, requests, tokens):
        pages = -(-tokens // PAGE)
        return [B.Kv4Cache(requests * pages, PAGE, HEADS, DIM, requests, pages) for _ in range(LAYERS)]

    def step(self, caches, new, tokens):
        """Logits of the new tokens (request after request), which stay in the caches."""
        x = self.embedding[tokens]
        for w, cache in zip(self.layers, caches):
            places = cache.step(new)
            assert places["unserved"] == 0, "the cache is full"
            qkv = B.mx4_linear(norm(x), w["qkv"]).reshape(len(x), -1, DIM)
            q, k, v = qkv[:, :QUERIES], qkv[:, QUERIES:-HEADS], qkv[:, -HEADS:]
            q = cache.append(k, v, q, self.turn)
            a, _ = cache.attend(q)
            x = x + B.mx4_linear(a.reshape(len(x), WIDTH), w["o"])
            x = x + B.mx4_linear(np.maximum(B.mx4_linear(norm(x), w["up"]), 0.0), w["down"])
        return B.mx4_linear(norm(x), self.head)


def norm(x):
    return x / np.sqrt((x * x).mean(1, keepdims=True) + 1e-6)


def generate(tokens=24, seed=0):
    """(the requests' tokens, the largest logit difference of prompts anew)."""
    rng = np.random.default_rng(seed)
    model = Model(seed)
    text = [list(rng.integers(0, VOCABULARY, n)) for n in (5, 33, 20)]
    caches = model.caches(len(text), 64 + tokens)
    new, going = [len(t) for t in text], [True] * len(text)
    logits = model.step(caches, new, np.concatenate(text))
    for i in range(tokens):
        last = np.cumsum([max(n, 0) for n in new]) - 1
        for r in range(len(text)):
            if going[r]:
                text[r].append(int(logits[last[r]].argmax()))
        new = [1 if g else 0 for g in going]
        if i == tokens // 2:
            new[1], going[1] = -1, False
        logits = model.step(caches, new, np.array([t[-1] for t, n in zip(text, new) if n > 0]))
    off = 0.0
    for row, r in enumerate(r for r in range(len(text)) if going[r]):
        anew = model.step(model.caches(1, len(text[r])), [len(text[r])], np.array(text[r]))
        off = max(off, float(np.abs(anew[-1] - logits[row]).max()))
    return text, off


if __name__ == "__main__":
    text, off = generate(int(sys.argv[1]) if len(sys.argv) > 1 else 24)
    for t in text:
        print(len(t), "tokens:", *t[-8:])
    print(f"logits of prompts anew: off by {off:.2g}")
    sys.exit(0 if off < 0.5 else "the logits differ")
