"""A paged cache built from plain per-sequence tensors, and attention over it
in 64 bits, for the tests of the paged operators."""

import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Paged:
    """`lens[b]` rows of sequence b (`news[b]` of them new) in shuffled pages.
    Rows of a page that hold nothing are NaN, and so are all pages of no
    sequence; table entries past a sequence's pages are not pages at all."""

    def __init__(self, news, lens, h, h_kv, d, page, dtype, token_major=False,
                 seed=0, spare=2, sharp=1.0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.news, self.lens, self.h, self.h_kv, self.d = news, lens, h, h_kv, d
        self.page, self.dtype = page, dtype
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)
        used = [-(-max(x, 0) // page) for x in lens]
        total, width = sum(used) + spare, max(max(used), 1)
        shape = (total, page, h_kv, d) if token_major else (total, h_kv, page, d)
        self.kp = torch.full(shape, float("nan"), device="cuda", dtype=dtype)
        self.vp = self.kp.clone()
        if token_major:
            self.kp, self.vp = self.kp.transpose(1, 2), self.vp.transpose(1, 2)
        order = torch.randperm(total, generator=g, device="cuda").tolist()
        table = torch.full((len(lens), width), 2 ** 30, dtype=torch.int32)
        for b, u in enumerate(used):
            for i in range(u):
                table[b, i] = order.pop()
        self.table = table.cuda()
        self.starts = torch.tensor([0] + news).cumsum(0).to(torch.int32).cuda()
        self.seq_lens = torch.tensor(lens, dtype=torch.int32).cuda()
        self.k = [rand(max(x, 0), h_kv, d) for x in lens]
        self.v = [rand(max(x, 0), h_kv, d) for x in lens]
        for b, n in enumerate(lens):
            for r0 in range(0, n, page):
                p, m = int(table[b, r0 // page]), min(page, n - r0)
                self.kp[p, :, :m] = self.k[b][r0:r0 + m].transpose(0, 1)
                self.vp[p, :, :m] = self.v[b][r0:r0 + m].transpose(0, 1)
        self.q = rand(sum(news), h, d) * sharp

    def exact(self, scale, causal=True):
        """64-bit output, each element's sum of p |v|, and the log-sum-exp."""
        t, g = sum(self.news), self.h // self.h_kv
        out = torch.zeros(t, self.h, self.d, dtype=torch.float64, device="cuda")
        size = torch.zeros_like(out)
        lse = torch.full((t, self.h), float("-inf"), dtype=torch.float64, device="cuda")
        lo = 0
        for b, n in enumerate(self.news):
            if n and self.lens[b] > 0:
                q = self.q[lo:lo + n].double().transpose(0, 1)
                k, v = (x[b].double().transpose(0, 1).repeat_interleave(g, 0)
                        for x in (self.k, self.v))
                s = q @ k.transpose(1, 2) * scale
                if causal:
                    row = torch.arange(self.lens[b] - n, self.lens[b], device="cuda")
                    key = torch.arange(self.lens[b], device="cuda")
                    s[:, key > row[:, None]] = float("-inf")
                z = torch.logsumexp(s, -1)
                p = torch.exp(s - torch.where(z.isfinite(), z, 0.0)[..., None])
                out[lo:lo + n] = (p @ v).transpose(0, 1)
                size[lo:lo + n] = (p @ v.abs()).transpose(0, 1)
                lse[lo:lo + n] = z.T
            lo += n
        return out, size, lse


def check_attention(c, got, scale, causal=True, lse=None):
    """Each probability enters the second product rounded to the 16-bit type
    (u of it at most), the result is rounded once more (u |o|), and the fp32
    scores and exponentials (the exponential itself is good to 8e-5) cost up
    to 5e-4 of sum p |v| for inputs of unit size."""
    want, size, want_lse = c.exact(scale, causal)
    u = UNIT[c.dtype]
    assert got.shape == c.q.shape and got.dtype == c.dtype
    err = (got.double() - want).abs()
    bad = ~(err <= (u + 5e-4) * size + u * want.abs() + 2.0 ** -25)
    assert not bool(bad.any()), (bad.nonzero()[:5].tolist(), err.max().item())
    if lse is not None:
        assert lse.dtype == torch.float32 and lse.shape == want_lse.shape
        empty = want_lse.isinf()
        assert torch.equal(lse.isinf() & (lse < 0), empty)
        assert bool(((lse.double() - want_lse).abs()[~empty] <= 5e-4).all())
