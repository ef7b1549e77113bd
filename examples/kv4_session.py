"""Sessions on a 4-bit KV cache, two ways.

``park``: a BaseLM session's fp16 cache (every layer of it) is put into 4 bits, 3.6 times smaller,
and brought back into an engine that goes on decoding.

``speculate``: a serving loop of several streams over one attention layer. Each round drafts a few
tokens, appends their K and V rows, attends with all of them in one pass, verifies them against the
model's probabilities, lets the next append overwrite what was rejected, and evicts the rows that
drew the least attention once a stream is over its budget. Nothing in the loop waits for the device.

    python examples/kv4_session.py
"""
import sys
import tempfile
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import numpy as np  # noqa: E402
import torch  # noqa: E402

from voxgen_b200 import kv4  # noqa: E402


def park(model_dir, preset="pin", prompt=48, more=8):
    """Decodes a prompt, parks the session, restores it and decodes on. Returns the largest difference of the hidden
    states against the session that was never parked, and the bytes of the two caches."""
    from voxgen_b200 import api, synth
    spec = synth.preset(preset)
    ctx = api.Context(0)
    model = api.Model(ctx, synth.model_path(spec, Path(model_dir)))
    info = model.info
    layers, heads, dim = info["block_count"], info["head_count_kv"], info["head_dim"]
    kept, restored = (api.BaseLmEngine(model, prompt + more) for _ in range(2))
    tokens = np.random.default_rng(7).integers(0, info["vocab_size"], prompt + more)
    kept.prefill_tokens(tokens[:prompt])

    # the layers are the sequences of one cache
    k, v = (torch.from_numpy(x.view(np.float16)).cuda().view(layers, prompt, heads, dim) for x in kept.read_kv(prompt))
    cache = kv4.Kv4Cache(layers, heads, dim, prompt)
    cache.append(k, v)
    if any(cache.status()):   # the engine's fp16 cache holds up to 65504, this one up to 7168
        raise ValueError("the session holds values that its 4-bit cache would clamp")

    back = [x.reshape(layers, prompt, heads * dim).cpu().numpy().view(np.uint16) for x in cache.read(prompt)]
    restored.write_kv(*back)
    worst = 0.0
    for t in tokens[prompt:]:
        for engine in (kept, restored):
            engine.decode_token_gpu_only(int(t))
        worst = max(worst, float(np.abs(kept.output() - restored.output()).max()))
    sizes = 4 * k.numel(), cache.data.numel()
    for x in (kept, restored, model, ctx):
        x.close()
    return worst, sizes


class Layer:
    """One attention layer between an embedding and a head, with random weights."""

    def __init__(self, seed=0, hidden=256, heads=8, kv_heads=2, head_dim=64, vocab=500):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def matrix(*shape):
            return torch.randn(*shape, generator=g, device="cuda") / shape[0] ** 0.5

        self.heads, self.kv_heads, self.head_dim, self.vocab = heads, kv_heads, head_dim, vocab
        self.embedding = torch.randn(vocab, hidden, generator=g, device="cuda")
        self.qkv = matrix(hidden, (heads + 2 * kv_heads) * head_dim)
        self.out, self.head = matrix(heads * head_dim, hidden), matrix(hidden, vocab) * 2

    def project(self, tokens):
        """q, k and v of tokens [streams, n], as views of one product."""
        x = self.embedding[tokens] @ self.qkv
        return x.unflatten(-1, (-1, self.head_dim)).split((self.heads, self.kv_heads, self.kv_heads), 2)

    def probabilities(self, tokens, attended):
        x = self.embedding[tokens] + attended.flatten(2) @ self.out
        return (x @ self.head).softmax(-1)

    def guess(self, tokens):
        """The draft's probabilities after tokens [streams]: the layer without its attention."""
        return (self.embedding[tokens] @ self.head).softmax(-1)


def speculate(streams=4, rounds=24, drafted=4, budget=48, recent=16, sinks=2, seed=0, attend=None):
    """Runs the loop; returns the emitted tokens [streams, rounds * (drafted + 1)], -1 where a draft was rejected, and
    the cache. ``attend(cache, q)`` stands in for the cache's own attention (for tests)."""
    layer = Layer(seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    room = budget + drafted + 1
    cache = kv4.Kv4Cache(streams, layer.kv_heads, layer.head_dim, room, track=True)
    attend = attend or (lambda c, q: c.attention(q))
    token = torch.randint(0, layer.vocab, (streams,), generator=g, device="cuda", dtype=torch.int32)
    rows = torch.zeros(streams, dtype=torch.int32, device="cuda")   # rows that hold accepted tokens
    place = torch.arange(drafted + 1, device="cuda")
    emitted = []
    for _ in range(rounds):
        u = torch.rand(streams, 2 * drafted + 1, generator=g, device="cuda")
        # draft: each token from the cheap model after the one before it
        run, guesses = [token], []
        for i in range(drafted):
            guesses.append(layer.guess(run[-1]))
            run.append((guesses[-1].cumsum(-1) < u[:, i:i + 1]).sum(-1).clamp_max(layer.vocab - 1).int())
        tokens = torch.stack(run, 1)                 # the last accepted token, then the drafts
        # the model, on all of them at once
        q, k, v = layer.project(tokens)
        cache.append(k, v, at=rows)
        target = layer.probabilities(tokens, attend(cache, q))
        accepted, token = kv4.verify_draft(tokens[:, 1:].contiguous(), torch.stack(guesses, 1), target,
                                           u[:, drafted:2 * drafted].contiguous(), u[:, -1].contiguous())
        # emitted: the accepted drafts and the token after them; the next append starts past the accepted rows
        run = torch.cat((tokens[:, 1:], token[:, None]), 1)
        run.scatter_(1, accepted[:, None].long(), token[:, None])
        emitted.append(torch.where(place <= accepted[:, None], run, -1))
        rows = rows + 1 + accepted
        cache.append(k[:, :1], v[:, :1], at=rows, counts=torch.zeros_like(rows))   # drops the rejected rows
        cache.evict(budget, recent, sinks)
        rows = cache.rows().clone()
    return torch.cat(emitted, 1), cache


def main():
    with tempfile.TemporaryDirectory() as d:
        worst, (half, four) = park(d)
    print(f"parked and restored: {half} bytes in fp16, {four} in 4 bits; hidden states differ by at most {worst:.3f}")
    tokens, cache = speculate()
    kept = (tokens >= 0).sum(1)
    print(f"speculated: {kept.tolist()} tokens in {tokens.shape[1] // 5} rounds, rows held {cache.rows().tolist()}")


if __name__ == "__main__":
    main()
