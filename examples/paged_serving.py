"""Requests that come, grow and finish on a paged KV cache.

``serve`` keeps a few slots busy: whenever a request has its tokens, its slot gives its pages back and, if
the pool will have room for all of it, takes the next request's prompt in the same step, so prompts and
single tokens share every launch. With ``budget`` the tokens attend over that many pages of their sequence, those that the selection picks.

    python examples/paged_serving.py
"""
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
sys.path.insert(0, str(Path(__file__).resolve().parent))

import torch  # noqa: E402

from kv4_session import Layer  # noqa: E402
from voxgen_b200.paged import PagedCache, PageTable  # noqa: E402


def serve(prompts, new=12, slots=4, page_rows=16, pages=64, budget=None, seed=0):
    """Greedy tokens after each prompt (lists of token numbers), ``new`` of them each, and the table at the end."""
    layer = Layer(seed)
    longest = max(map(len, prompts)) + new
    table = PageTable(slots, pages, page_rows, -(-longest // page_rows))
    cache = PagedCache(table, layer.kv_heads, layer.head_dim, summaries=budget is not None)
    waiting, answers = list(enumerate(prompts)), [[] for _ in prompts]
    running = [None] * slots                 # the request of each slot
    fresh = [[] for _ in range(slots)]       # tokens that a slot's request has not stored yet

    def most(r):                             # pages that a request takes in the end
        return -(-(len(prompts[r]) + new) // page_rows)

    assert max(most(r) for r in range(len(prompts))) <= pages
    while waiting or any(r is not None for r in running):
        keep = [-1] * slots
        for s, r in enumerate(running):
            if r is None or len(answers[r]) == new:
                keep[s], running[s], fresh[s] = 0, None, []      # its pages are free within this step
        for s, r in enumerate(running):
            if r is None and waiting and sum(most(x) for x in running if x is not None) + most(waiting[0][0]) <= pages:
                running[s], prompt = waiting.pop(0)
                fresh[s] = list(prompt)
        counts = torch.tensor([len(x) for x in fresh], dtype=torch.int32, device="cuda")
        tokens = torch.tensor(sum(fresh, []), dtype=torch.int32, device="cuda")
        step = table.step(counts, len(tokens), keep=torch.tensor(keep, dtype=torch.int32, device="cuda"))
        if not len(tokens):
            break
        q, k, v = (x[0] for x in layer.project(tokens[None]))
        cache.append(step, k, v)
        which = dict(sequences=step.sequences, positions=step.positions)
        if budget is not None:
            which["chosen"] = cache.select(q, budget, sinks=1, recent=1, **which)
        attended = cache.attention(q, **which)
        last = step.starts[1:].clamp_min(1).long() - 1           # of each slot's tokens
        best = layer.probabilities(tokens[last][:, None], attended[last][:, None])[:, 0].argmax(-1).tolist()
        assert not table.status.any()
        for s, r in enumerate(running):
            if r is not None:
                answers[r].append(best[s])
                fresh[s] = [best[s]]
    return answers, table


def main():
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 500, (int(n),), generator=g).tolist() for n in torch.randint(3, 90, (10,), generator=g)]
    answers, table = serve(prompts)
    few, _ = serve(prompts, budget=3)
    same = sum(a == b for x, y in zip(answers, few) for a, b in zip(x, y))
    print(f"{len(answers)} requests of {len(answers[0])} tokens; {int(table.pool[0])} of {table.pages} pages free at the end; "
          f"with 3 pages a token {same} of {sum(map(len, answers))} tokens are the same")


if __name__ == "__main__":
    main()
