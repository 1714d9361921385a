"""One attention layer trained a little, then served over a guarded 8-bit paged cache.

    python examples/guarded_decode.py [--tokens 48] [--cache e4m3|int8]

The queries and keys of a layer are rotated by position with their gradient (rope.rotate) for a few training steps.  The
trained layer then serves two sequences: their prompts as chunks, the rest token by token.  Each step verifies the pages
that earlier steps wrote, codes and scales (a KVLedger each), appends its keys and values, rotated and quantized on the way
(kv_attn.kv_append), attends over the cache (kv_attn.kv_attend) and records the pages it changed.  At the end the outputs are
compared with the layer's 16-bit attention, and one flipped bit of the codes and one of the scales have to be found.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from sdcguard_amd import frequencies, kv_append, kv_attend, make_cache, rotate  # noqa: E402
from sdcguard_amd.kv import KVLedger  # noqa: E402

HEADS, KV_HEADS, DIM, SLOTS = 8, 2, 64, 16
CACHES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def plain_attention(q, k, v):
    """Causal attention of (tokens, heads, head size) in fp32, kv heads shared by groups of query heads."""
    k, v = (t.float().repeat_interleave(q.shape[1] // t.shape[1], 1).transpose(0, 1) for t in (k, v))
    s = (q.float().transpose(0, 1) @ k.transpose(1, 2)) * q.shape[2] ** -0.5
    n = q.shape[0]
    s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), float("-inf"))
    return (torch.softmax(s, -1) @ v).transpose(0, 1)


class Layer:
    def __init__(self, width, turns, mscale, device):
        g = torch.Generator(device=device).manual_seed(1)
        out = (HEADS + 2 * KV_HEADS) * DIM
        self.w = (torch.randn(out, width, generator=g, device=device) * width ** -0.5).requires_grad_()
        self.turns, self.mscale = turns, mscale

    def project(self, x):
        qkv = (x @ self.w.t()).bfloat16()
        return (t.unflatten(-1, (-1, DIM)) for t in qkv.split([HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM], -1))

    def attend(self, x):
        """The layer on whole sequences, as it is trained."""
        q, k, v = self.project(x)
        pos = torch.arange(x.shape[0], device=x.device)
        q, k = (rotate(t, pos, self.turns, mscale=self.mscale) for t in (q, k))
        return plain_attention(q, k, v)


def train(layer, x, steps=3, rate=0.05):
    """A few steps towards outputs that copy the previous token's first features; the losses."""
    want = torch.roll(x[:, :HEADS * DIM], 1, 0).reshape(-1, HEADS, DIM).detach()
    losses = []
    for _ in range(steps if x.shape[0] > 1 else 0):             # (one token has no other to copy)
        loss = (layer.attend(x)[1:] - want[1:]).square().mean()
        grad, = torch.autograd.grad(loss, layer.w)
        with torch.no_grad():
            layer.w -= rate * grad / grad.square().mean().sqrt() * layer.w.square().mean().sqrt()
        losses.append(loss.item())
    return losses


def serve(layer, xs, prompt, cache):
    """The sequences' outputs, served over a paged cache: (outputs, cache, scales, table, ledgers, mismatched pages)."""
    dev, R, n = xs[0].device, len(xs), xs[0].shape[0]
    width = -(-n // SLOTS)
    kv, scales = make_cache(R * width + 1, KV_HEADS, SLOTS, DIM, CACHES[cache], dev)
    order = torch.randperm(R * width, generator=torch.Generator().manual_seed(2)).to(torch.int32)
    table = (order + 1).view(R, width).to(dev)                   # page 0 stays empty
    # (a scale multiplies a whole page of a head: unguarded, one flipped bit of it would go unseen)
    ledgers = KVLedger(kv.view(torch.uint8), R, width), KVLedger(scales, R, width)
    outs, bad, at = [[] for _ in xs], 0, 0
    column = torch.arange(width, device=dev)
    with torch.no_grad():
        while at < n:
            new = prompt if at == 0 else 1
            x = torch.cat([s[at:at + new] for s in xs])
            qsl = torch.arange(R + 1, device=dev, dtype=torch.int32) * new
            lens = torch.full((R,), at + new, device=dev, dtype=torch.int32)
            bad += sum(int(ledger.verify(table).count) for ledger in ledgers)
            q, k, v = layer.project(x)
            q = kv_append(k, v, kv, scales, qsl, lens, table, turns=layer.turns, mscale=layer.mscale, query=q)
            o = kv_attend(q, kv, scales, qsl, lens, table, max_seq_len=n)
            written = (column >= at // SLOTS) & (column <= (at + new - 1) // SLOTS)
            for ledger in ledgers:
                ledger.record(table, written.expand(R, width))
            for r in range(R):
                outs[r].append(o[r * new:(r + 1) * new])
            at += new
    return [torch.cat(o) for o in outs], kv, scales, table, ledgers, bad


def main(tokens=48, cache="e4m3", quiet=False):
    dev = torch.device("cuda", torch.cuda.current_device())
    turns, mscale = frequencies(DIM, 500000.0, {"kind": "ramp", "factor": 4.0, "trained": 1024}, dev)
    layer = Layer(HEADS * DIM, turns, mscale, dev)
    g = torch.Generator(device=dev).manual_seed(3)
    xs = [torch.randn(tokens, HEADS * DIM, generator=g, device=dev) for _ in range(2)]
    losses = train(layer, xs[0])
    outs, kv, scales, table, (codes_ledger, scales_ledger), bad = serve(layer, xs, max(1, tokens // 2), cache)
    with torch.no_grad():
        wants = [layer.attend(x) for x in xs]
    off = max(float((o.float() - w).abs().max() / w.abs().max()) for o, w in zip(outs, wants))
    kv.view(torch.uint8)[table[1, 0].long(), 0, 3, 5] ^= 4        # one flipped bit of a code, one of a scale's exponent
    scales.view(torch.int32)[table[0, 0].long(), 1, 0] ^= 1 << 24
    found = codes_ledger.verify(table).read()
    found["scale_entries"] = scales_ledger.verify(table).read()["entries"]
    if not quiet:
        print(f"loss {' -> '.join(f'{x:.4f}' for x in losses)}; {tokens} tokens over a {cache} cache: off by {off:.3f} of the "
              f"largest output; pages changed unseen: {bad}; after a flipped bit of the codes: {found['entries']}, of the scales: {found['scale_entries']}")
    return losses, off, bad, found


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--tokens", type=int, default=48)
    p.add_argument("--cache", choices=sorted(CACHES), default="e4m3")
    a = p.parse_args()
    main(a.tokens, a.cache)
