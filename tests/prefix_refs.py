"""Batches of requests that share pages, and their attention in 64 bits, for the tests of shared prefixes."""
import torch


class Batch:
    """A tree of prefixes.  `tree`: (tokens shared, [children]) with leaves (own tokens before the new ones, new tokens); shared tokens are whole pages."""

    def __init__(self, tree, nq, nkv, hd, vd, ps, seed=0, dtype=torch.float32, spare=3, strided=8):
        g = torch.Generator().manual_seed(seed)
        self.nq, self.nkv, self.hd, self.vd, self.ps = nq, nkv, hd, vd, ps
        self.tables, self.q_lens, self.ctx_lens, free, held = [], [], [], iter(range(10 ** 6)), set()

        def walk(node, front):
            tokens, rest = node
            if isinstance(rest, list):
                assert tokens % ps == 0
                pages = front + [next(free) for _ in range(tokens // ps)]
                for child in rest:
                    walk(child, pages)
            else:
                ctx = len(front) * ps + tokens + rest
                self.tables.append(front + [next(free) for _ in range(-(-ctx // ps) - len(front))])
                self.q_lens.append(rest)
                self.ctx_lens.append(ctx)
        walk(tree, [])
        self.R, self.n = len(self.q_lens), sum(self.q_lens)
        used = next(free)
        order = torch.randperm(used + spare, generator=g).tolist()
        width = max(len(t) for t in self.tables) + 2
        self.table = torch.full((self.R, width), -1, dtype=torch.int32)
        for r, t in enumerate(self.tables):
            self.table[r, :len(t)] = torch.tensor([order[p] for p in t], dtype=torch.int32)
        # slots that hold no token of anybody hold no numbers
        self.k, self.v = (torch.full((used + spare, nkv, ps, d), float("nan")) for d in (hd, vd))
        for r, ctx in enumerate(self.ctx_lens):
            for i in range(-(-ctx // ps)):
                page = int(self.table[r, i])
                n = min(ps, ctx - i * ps)
                if page not in held:
                    held.add(page)
                    self.k[page, :, :n], self.v[page, :, :n] = torch.randn(nkv, n, hd, generator=g), torch.randn(nkv, n, vd, generator=g)
        wide = torch.randn(self.n, nq * hd + strided, generator=g) * 2
        self.sinks, self.slopes = torch.randn(nq, generator=g), torch.rand(nq, generator=g) * 0.2
        self.k, self.v, wide = (t.to(dtype) for t in (self.k, self.v, wide))
        self.q = wide[:, :nq * hd]

    def exact(self, scale, sinks=None, cap=0.0, slopes=None):
        """[tokens, nq * vd] in 64 bits, request by request."""
        out, start, rep = torch.empty(self.n, self.nq * self.vd, dtype=torch.float64), 0, self.nq // self.nkv
        for r, (n, ctx) in enumerate(zip(self.q_lens, self.ctx_lens)):
            pages = self.table[r, :-(-ctx // self.ps)].long()
            k, v = (t[pages].double().transpose(1, 2).reshape(-1, self.nkv, t.shape[-1])[:ctx].repeat_interleave(rep, 1) for t in (self.k, self.v))
            q = self.q[start:start + n].double().view(n, self.nq, self.hd)
            s = torch.einsum("nhd,khd->nhk", q, k) * scale
            if cap:
                s = cap * torch.tanh(s / cap)
            away = (torch.arange(ctx - n, ctx)[:, None] - torch.arange(ctx)[None, :])[:, None, :]
            if slopes is not None:
                s = s - slopes.double()[None, :, None] * away
            s = s.masked_fill(away < 0, float("-inf"))
            if sinks is not None:
                s = torch.cat([s, sinks.double()[None, :, None].expand(n, -1, 1)], -1)
            w = torch.softmax(s, -1)[..., :ctx]
            out[start:start + n] = torch.einsum("nhk,khd->nhd", w, v).reshape(n, -1)
            start += n
        return out

    def on(self, device):
        """(q, key pages, value pages, block table) on the device, q with its row stride."""
        wide = torch.empty(self.n, self.q.stride(0), dtype=self.q.dtype, device=device)
        q = wide[:, :self.q.shape[1]]
        q.copy_(self.q)
        return q, self.k.to(device), self.v.to(device), self.table.to(device)
