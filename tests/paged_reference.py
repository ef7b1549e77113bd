"""The paged cache's operators in Python and 64-bit arithmetic, for the tests: written from their
definitions, apart from the kernels and from the forms that the benchmark compares with."""
import numpy as np
import torch

FULL, NO_PAGES, BAD_COUNT = 1, 2, 4


class Table:
    """The state of a page table, one sequence after another."""

    def __init__(self, seqs, pages, page_rows, seq_pages, free=None):
        self.page, self.most = page_rows, seq_pages
        self.held = [[] for _ in range(seqs)]       # pages of each sequence
        self.rows = [0] * seqs
        self.status = [0] * seqs
        self.free = list(range(pages)) if free is None else list(free)

    def step(self, counts, tokens, keep=None):
        """starts, slots, positions, sequences, runs of one step."""
        page, n = self.page, len(self.rows)

        def pages_of(rows):
            return -(-rows // page)

        kept = [r if keep is None or keep[s] < 0 else min(r, keep[s]) for s, r in enumerate(self.rows)]
        for s in range(n):
            self.free += self.held[s][pages_of(kept[s]):]
            self.held[s] = self.held[s][:pages_of(kept[s])]
        starts, demand, need, fresh = [], 0, [0] * n, [0] * n
        total = 0
        for s, c in enumerate(counts):
            starts.append(min(total, tokens))
            self.status[s] = 0
            if not 0 <= c <= tokens:
                self.status[s] = BAD_COUNT
                continue
            total += c
            if total > tokens:
                self.status[s] = BAD_COUNT
            elif kept[s] + c > self.most * page:
                self.status[s] = FULL
            else:
                want = pages_of(kept[s] + c) - pages_of(kept[s])
                demand += want
                if want and demand > len(self.free):
                    self.status[s] = NO_PAGES
                else:
                    need[s], fresh[s] = want, c
        starts.append(min(total, tokens))
        top = len(self.free) - sum(need)
        taken, self.free = self.free[top:], self.free[:top]
        slots, positions, sequences, runs = [-1] * tokens, [-1] * tokens, [-1] * tokens, []
        for s in range(n):
            self.held[s] += taken[:need[s]]
            taken = taken[need[s]:]
            self.rows[s] = kept[s] + fresh[s]
            for i in range(fresh[s]):
                p = kept[s] + i
                t = starts[s] + i
                slots[t], positions[t], sequences[t] = self.held[s][p // page] * page + p % page, p, s
                if i == 0 or p % page == 0:
                    runs.append([t, self.held[s][p // page], p % page, 0])
                runs[-1][3] += 1
        most = min(tokens, tokens // page + 2 * n)
        assert len(runs) <= most
        runs += [[0, 0, 0, 0]] * (most - len(runs))
        return starts, slots, positions, sequences, runs

    def table(self):
        return [h + [-1] * (self.most - len(h)) for h in self.held]


def attention(q, k, v, rows, scale=None):
    """One query's heads [heads, head_dim] over the rows k, v [kv_heads, rows, head_dim] in 64 bits (torch, on any device);
    rows: which of them each KV head attends, row numbers a head."""
    heads, dim = q.shape
    group = heads // k.shape[0]
    out = torch.zeros(heads, dim, dtype=torch.float64, device=q.device)
    for h, mine in enumerate(rows):
        if len(mine):
            e = q[h * group:(h + 1) * group].double() @ k[h, mine].T * (dim ** -0.5 if scale is None else scale)
            p = (e - e.amax(1, keepdim=True)).exp()
            out[h * group:(h + 1) * group] = p / p.sum(1, keepdim=True) @ v[h, mine]
    return out


def choose(q, low, high, budget, sinks, recent):
    """Pages that the heads q [group, head_dim] choose, given the extremes [pages, head_dim] of each page."""
    n = len(low)
    if n <= budget:
        return list(range(n)) + [-1] * (budget - n)
    q = np.nan_to_num(q.astype(np.float64), nan=0.0, posinf=3.402823466e38, neginf=-3.402823466e38)
    score = np.maximum(q[:, None] * low, q[:, None] * high).sum((0, 2))
    sure = set(range(sinks)) | set(range(n - recent, n))
    rest = sorted((r for r in range(n) if r not in sure), key=lambda r: (-score[r], r))
    return sorted(sure | set(rest[:budget - len(sure)]))
