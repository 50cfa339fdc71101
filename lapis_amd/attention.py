"""Block-sparse attention over CSR structures, put together: training or prefill over chosen blocks of keys, and decoding
over the pages of a cache.

``choose_blocks``   8-bit means of the blocks of queries and keys, and the best blocks of keys to each as a CSR structure
``attend``          attention over such a structure, differentiable in q, k and v
``PagedCache``      keys and values in pages: ``prefill`` a sequence, ``step`` all of them by one token

``python -m lapis_amd.attention`` trains one layer to look values up in a long sequence, then answers from a cache token by
token.  Tensors are torch CUDA tensors of bfloat16 or float16: q is batch x queries x heads x dim, k and v are batch x keys x
key-value heads x dim.
"""
from dataclasses import dataclass

import torch

from . import hip


@dataclass
class Blocks:
    """A CSR structure: row (batch entry, key-value head, block of ``block_m`` queries) lists blocks of ``block_n`` keys."""
    pos: torch.Tensor
    crd: torch.Tensor
    block_m: int
    block_n: int
    causal: bool


def _means(x, block, groups):
    """Codes and scales of the means of x (batch x tokens x heads x dim) over ``block`` tokens and the heads of each group."""
    batch, tokens, _, dim = x.shape
    blocks = -(-tokens // block)
    codes = torch.empty((batch, groups, blocks, dim), dtype=torch.int8, device=x.device)
    scales = torch.empty((batch, groups, blocks), device=x.device)
    hip.block_pool(x, block, codes, scales)
    return codes, scales


def choose_blocks(q, k, count, block_m=64, block_n=64, causal=True, sink=1, local=2):
    """The ``count`` blocks of keys whose mean answers best to the mean of each block of queries; the first ``sink`` and the
    last ``local`` blocks that it may see are always among them."""
    batch, queries, _, _ = q.shape
    keys, groups = k.shape[1:3]
    q_codes, _ = _means(q.detach(), block_m, groups)
    k_codes, k_scales = _means(k.detach(), block_n, groups)
    rows, columns = q_codes.shape[2], k_codes.shape[2]
    pos = torch.empty(batch * groups * rows + 1, dtype=torch.int32, device=q.device)
    crd = torch.zeros(batch * groups * rows * min(count, columns), dtype=torch.int32, device=q.device)
    hip.block_select(q_codes, k_codes, k_scales, count, pos, crd, queries, keys, block_m, block_n, causal, sink, local)
    return Blocks(pos, crd, block_m, block_n, causal)


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, blocks, scale):
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), device=q.device)
        hip.block_attention(q, k, v, blocks.pos, blocks.crd, out, lse, blocks.block_m, blocks.block_n, blocks.causal, scale)
        ctx.save_for_backward(q, k, v, out, lse, blocks.pos, blocks.crd)
        ctx.sizes = blocks.block_m, blocks.block_n, blocks.causal, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable  # the gradient has none itself: asked for one it raises
    def backward(ctx, dout):
        q, k, v, out, lse, pos, crd = ctx.saved_tensors
        dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v))
        hip.block_attention_backward(dout.contiguous(), q, k, v, out, lse, pos, crd, dq, dk, dv, *ctx.sizes)
        return dq, dk, dv, None, None


def attend(q, k, v, blocks, scale=None):
    """softmax(scale q k^T) v over the listed blocks only; ``scale`` defaults to dim ** -0.5."""
    return _Attend.apply(q, k, v, blocks, scale)


class PagedCache:
    """Keys and values of ``sequences`` sequences in pages, with the 8-bit mean of each full page.  ``dtype`` is that of the
    rows that come in; with ``f8`` the cache holds them as e4m3 codes with a scale each."""

    def __init__(self, sequences, pages, longest, heads, dim, page=64, dtype=torch.bfloat16, f8=False, device="cuda"):
        kept = torch.float8_e4m3fn if f8 else dtype
        self.page, self.dtype = page, dtype
        self.k, self.v = (torch.zeros((pages, heads, page, dim), dtype=dtype, device=device).to(kept) for _ in range(2))
        self.k_scale, self.v_scale = (torch.zeros((pages, heads, page), device=device) if f8 else None for _ in range(2))
        self.codes = torch.zeros((pages, heads, dim), dtype=torch.int8, device=device)
        self.scales = torch.zeros((pages, heads), device=device)
        self.table = torch.zeros((sequences, -(-longest // page)), dtype=torch.int32, device=device)
        self.length = torch.zeros(sequences, dtype=torch.int32, device=device)
        self.lengths = [0] * sequences  # the same numbers on the host, which gives out the pages
        self.held = [[] for _ in range(sequences)]
        self.free = list(range(pages))[::-1]

    def _open(self, sequences, tokens):
        """Pages for ``tokens`` more tokens of each of these sequences; raises before anything changes where there are not enough."""
        free, needed = len(self.free), []
        for s in sequences:
            held = len(self.held[s])
            needed.append(max(0, -(-(self.lengths[s] + tokens) // self.page) - held))
            if needed[-1] > free or held + needed[-1] > self.table.shape[1]:
                raise RuntimeError("PagedCache: %d more pages for sequence %d, %d are free, %d of %d held" % (
                    needed[-1], s, free, held, self.table.shape[1]))
            free -= needed[-1]
        for s, n in zip(sequences, needed):
            new = [self.free.pop() for _ in range(n)]
            if new:
                first = len(self.held[s])
                self.table[s, first:first + n] = torch.tensor(new, dtype=torch.int32).to(self.table.device)
            self.held[s] += new

    def _store(self, k, v, slots):
        hip.kv_store(k, v, slots, self.k, self.v, self.k_scale, self.v_scale)

    def _keep_means(self, pages, k):
        """k: pages x page x heads x dim."""
        codes, scales = _means(k, self.page, k.shape[2])
        self.codes[pages], self.scales[pages] = codes[:, :, 0], scales[:, :, 0]

    def prefill(self, sequence, k, v):
        """The tokens (k, v: tokens x heads x dim) of an empty sequence."""
        if self.lengths[sequence]:
            raise ValueError("PagedCache.prefill: sequence %d holds %d tokens" % (sequence, self.lengths[sequence]))
        tokens, page = k.shape[0], self.page
        self._open([sequence], tokens)
        t = torch.arange(tokens, device=k.device)
        slots = self.table[sequence][t // page] * page + t % page
        self._store(k, v, slots.to(torch.int32))
        full = tokens // page
        if full:
            self._keep_means(self.table[sequence, :full].long(), k[:full * page].reshape(full, page, *k.shape[1:]))
        self.length[sequence] = self.lengths[sequence] = tokens

    def release(self, sequence):
        """Gives the pages of a sequence back."""
        self.free += self.held[sequence][::-1]
        self.held[sequence] = []
        self.length[sequence] = self.lengths[sequence] = 0

    def step(self, q, k, v, count, sink=1, local=2, scale=None):
        """One token more of every sequence (k, v: sequences x heads x dim), and what it reads (q: sequences x query heads x
        dim) from the ``count`` best pages of each sequence and key-value head; the last ``local`` (at least 1) and first
        ``sink`` pages are always among them.  A sequence that was released begins anew with its token.  Where the call raises, the
        cache holds what it held before."""
        if local < 1:
            raise ValueError("PagedCache.step: the page of the token itself is always attended to: local = %d" % local)
        if sink < 0 or count < sink + local:
            raise ValueError("PagedCache.step: %d pages, the first %d and the last %d always among them" % (count, sink, local))
        page, sequences, groups = self.page, len(self.lengths), self.k.shape[1]
        q_codes, _ = _means(q[:, None], 1, groups)
        self._open(range(sequences), 1)
        at = self.table.gather(1, (self.length // page).long()[:, None])[:, 0]
        self._store(k, v, at * page + self.length % page)
        # the numbers of the cache itself change when all is done: what was written counts from then on
        length, lengths = self.length + 1, [n + 1 for n in self.lengths]
        if any(n % page == 0 for n in lengths):  # pages that are full now
            pages = torch.tensor([self.held[s][n // page - 1] for s, n in enumerate(lengths) if n % page == 0], device=q.device)
            slots = (pages[:, None] * page + torch.arange(page, device=q.device)).to(torch.int32).reshape(-1)
            rows, unused = (torch.empty((slots.numel(), groups, q.shape[2]), dtype=self.dtype, device=q.device) for _ in range(2))
            hip.kv_load(self.k, self.v, slots, rows, unused, self.k_scale, self.v_scale)
            self._keep_means(pages, rows.reshape(-1, page, *rows.shape[1:]))

        blocks = (length + (page - 1)) // page
        pos = torch.empty(sequences * groups + 1, dtype=torch.int32, device=q.device)
        crd = torch.zeros(sequences * groups * min(count, self.table.shape[1]), dtype=torch.int32, device=q.device)
        hip.block_select(q_codes, self.codes, self.scales, count, pos, crd, 1, self.table.shape[1], 1, 1, False, sink, local,
                         self.table, blocks)
        # of the listed pages the last is the one the token is in
        tokens = (blocks.clamp(max=count) * page - (blocks * page - length)).repeat_interleave(groups)
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        hip.paged_attention(q, self.k, self.v, pos, crd, tokens, out, None, scale, self.k_scale, self.v_scale)
        self.length.copy_(length)
        self.lengths = lengths
        return out


def main(tokens=4096, asked=512, steps=100, heads=4, kv_heads=2, dim=64, block=16, count=24, seed=0, log=print):
    """Tokens carry a name and a value, and neighbours have names alike; the last ``asked`` tokens carry the name of an earlier
    one and are to answer its value.  Trains the projections over chosen blocks, on other tokens in each step, then prefills a
    cache and answers token by token.  Returns the losses of the steps, the mean square difference of answers from all pages
    to those of one pass over all blocks, and the loss of answers from ``count`` pages."""
    hip.init()
    g = torch.Generator().manual_seed(seed)
    every = -(-tokens // block)

    def sample():
        topics = torch.randn((every, dim), generator=g).repeat_interleave(block, 0)[:tokens]
        names, values = topics + torch.randn((tokens, dim), generator=g), torch.randn((tokens, dim), generator=g)
        where = torch.randint(0, tokens - asked, (asked,), generator=g).sort().values
        target = values[where].cuda()
        names[-asked:], values[-asked:] = names[where], 0.0
        return torch.cat([names, values], 1).cuda(), target

    weights = [(torch.randn(s, generator=g) * s[0] ** -0.5).cuda() for s in (
        (2 * dim, kv_heads * dim), (2 * dim, kv_heads * dim), (heads * dim, dim))]
    # queries and keys begin alike
    weights.insert(0, weights[0].view(2 * dim, kv_heads, dim).repeat_interleave(heads // kv_heads, 1).reshape(2 * dim, -1).clone())
    for w in weights:
        w.requires_grad_()
    adam = torch.optim.Adam(weights, 1e-2)

    def project(x):
        return ((x @ w).to(torch.bfloat16).view(1, tokens, -1, dim) for w in weights[:3])

    losses = []
    for step in range(steps):
        x, target = sample()
        q, k, v = project(x)
        out = attend(q, k, v, choose_blocks(q, k, count, block, block))
        loss = torch.nn.functional.mse_loss((out.view(tokens, -1).float() @ weights[3])[-asked:], target)
        adam.zero_grad()
        loss.backward()
        adam.step()
        losses.append(loss.item())
        if step % 10 == 0 or step == steps - 1:
            log("step %3d  loss %.4f" % (step, losses[-1]))

    with torch.no_grad():
        x, target = sample()
        q, k, v = project(x)
        whole = attend(q, k, v, choose_blocks(q, k, every, block, block))[0, -asked:].float()
        loss_of = lambda answers: torch.nn.functional.mse_loss(answers.reshape(asked, -1).float() @ weights[3], target).item()  # noqa: E731
        cache = PagedCache(1, every, tokens, kv_heads, dim, block)

        def answer(pages):
            cache.release(0)
            cache.prefill(0, k[0, :-asked], v[0, :-asked])
            return torch.cat([cache.step(q[0, t:t + 1], k[0, t:t + 1], v[0, t:t + 1], pages) for t in range(tokens - asked, tokens)])

        difference = (answer(every).float() - whole).square().mean().item()
        answered = loss_of(answer(count))
        log("all %d blocks in one pass: loss %.4f; token by token: mean square difference %.3g" % (every, loss_of(whole), difference))
        log("token by token from %d pages: loss %.4f" % (count, answered))
    return losses, difference, answered


if __name__ == "__main__":
    main()
