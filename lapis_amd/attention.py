"""Block-sparse attention over CSR structures, put together: training or prefill over chosen blocks of keys or over windows, and
decoding over the pages of a cache.

``choose_blocks``   8-bit means of the blocks of queries and keys, and the best blocks of keys to each as a CSR structure
``attend``          attention over such a structure, differentiable in q, k and v
``rotate``          queries or keys turned by the positions of their tokens, differentiable
``attend_window``   attention over the last keys of each query and the first ones, differentiable in q, k and v
``PagedCache``      keys and values in pages: ``prefill`` a sequence, ``step`` or ``step_window`` all of them by one token

``python -m lapis_amd.attention`` trains one layer to look values up in a long sequence, then answers from a cache token by
token.  Tensors are torch CUDA tensors of bfloat16 or float16: q is batch x queries x heads x dim, k and v are batch x keys x
key-value heads x dim.

A backward pass may be captured into a graph with the forward pass it belongs to.  As for all of torch's: no graph of autograd that was
made outside of the capture may still live on the same leaves, or the process ends; drop its tensors first.
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


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, frequencies, neighbours):
        ctx.save_for_backward(positions, frequencies)
        ctx.neighbours = neighbours
        return hip.rotate(x, positions, frequencies, torch.empty(x.shape, dtype=x.dtype, device=x.device), neighbours)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        dout = dout.contiguous()  # a broadcast one has strides that the kernel would take, but not every dout has
        return hip.rotate(dout, *ctx.saved_tensors, torch.empty_like(dout), ctx.neighbours, True), None, None, None


def rotate(x, positions, frequencies, neighbours=False):
    """Queries or keys (x: batch x tokens x heads x dim) turned by their ``positions`` (axes x batch x tokens, int32) times
    ``frequencies`` (axes x pairs, float64): elements i and i + pairs, or with ``neighbours`` 2i and 2i + 1.  Differentiable in x."""
    return _Rotate.apply(x, positions, frequencies, neighbours)


def _near(q, kv_heads):
    """q as the gradient of windows takes it: its tokens and heads less than 2 ** 25 elements apart, and 63 tokens and a group's heads
    within 2 ** 31.  The forward pass takes any."""
    token, head = (q.stride(i) if q.shape[i] > 1 else 0 for i in (1, 2))
    group = max(q.shape[2] // kv_heads, 1)
    near = max(token, head) < 2 ** 25 and (62 // group + 1) * token + (group - 1) * head + 128 < 2 ** 31
    return q if near else q.contiguous()


class _AttendWindow(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sink, scale):
        group = q.shape[2] // max(k.shape[2], 1)
        if any(ctx.needs_input_grad) and q.shape[1] * group >= 2 ** 29:
            raise ValueError("attend_window: a gradient of %d queries of %d heads of a group, fewer than 2 ** 29 together expected" % (q.shape[1], group))
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), device=q.device)
        hip.window_attention(q, k, v, out, window, sink, lse, scale)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.sizes = window, sink, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v))
        hip.window_attention_backward(dout.contiguous(), _near(q, k.shape[2]), k, v, out, lse, dq, dk, dv, *ctx.sizes)
        return dq, dk, dv, None, None, None


def attend_window(q, k, v, window, sink=0, scale=None):
    """softmax(scale q k^T) v where a query, the last of which stands at the last key, sees the last ``window`` keys up to its own and
    the first ``sink``; ``scale`` defaults to dim ** -0.5."""
    return _AttendWindow.apply(q, k, v, window, sink, scale)


class PagedCache:
    """Keys and values of ``sequences`` sequences in pages, with the 8-bit mean of each full page.  ``dtype`` is that of the
    rows that come in; with ``f8`` the cache holds them as e4m3 codes with a scale each, with ``f4`` as codes of 4 bits with a power of
    two for each 32 elements.  With ``frequencies`` (and ``neighbours``, as of ``rotate``) the queries and keys that come in are turned by the
    positions of their tokens: by ``positions`` (axes x tokens, int32) where a call is given them, else by the numbers of the tokens in their
    sequences on every axis."""

    def __init__(self, sequences, pages, longest, heads, dim, page=64, dtype=torch.bfloat16, f8=False, device="cuda", f4=False,
                 frequencies=None, neighbours=False):
        if f8 and f4:
            raise ValueError("PagedCache: codes of 8 bits and of 4 bits")
        if f4 and dim % 32:
            raise ValueError("PagedCache: rows of %d elements, of which each 32 have a scale" % dim)
        kept, row, scales = (torch.uint8, dim // 2, (dim // 32,)) if f4 else (torch.float8_e4m3fn if f8 else dtype, dim, ())
        self.page, self.dtype, self.frequencies, self.neighbours = page, dtype, frequencies, neighbours
        self.k, self.v = (torch.zeros((pages, heads, page, row), dtype=dtype, device=device).to(kept) for _ in range(2))
        self.k_scale, self.v_scale = (
            torch.zeros((pages, heads, page) + scales, dtype=torch.uint8 if f4 else torch.float32, device=device) if f8 or f4 else None
            for _ in range(2))
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

    def _store(self, q, k, v, slots, numbers, positions):
        """Into ``slots``; tokens of these numbers in their sequences.  Returns q as it is used (None if there is none)."""
        if self.frequencies is None:
            hip.kv_store(k, v, slots, self.k, self.v, self.k_scale, self.v_scale)
            return q
        if positions is None:
            positions = numbers.to(torch.int32).expand(self.frequencies.shape[0], -1)
        turned = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
        hip.kv_append(k, v, positions, self.frequencies, slots, self.k, self.v, self.k_scale, self.v_scale, q, turned, self.neighbours)
        return turned

    def _keep_means(self, pages, k=None):
        """k: pages x page x heads x dim; without it the keys are read back."""
        if k is None:
            slots = (pages[:, None] * self.page + torch.arange(self.page, device=pages.device)).to(torch.int32).reshape(-1)
            rows, unused = (torch.empty((slots.numel(), self.k.shape[1], self.codes.shape[2]), dtype=self.dtype, device=pages.device)
                            for _ in range(2))
            hip.kv_load(self.k, self.v, slots, rows, unused, self.k_scale, self.v_scale)
            k = rows.reshape(-1, self.page, *rows.shape[1:])
        codes, scales = _means(k, self.page, k.shape[2])
        self.codes[pages], self.scales[pages] = codes[:, :, 0], scales[:, :, 0]

    def _check_positions(self, what, positions):
        if positions is not None and self.frequencies is None:
            raise ValueError("PagedCache.%s: positions, and no frequencies" % what)

    def prefill(self, sequence, k, v, q=None, positions=None):
        """The tokens (k, v: tokens x heads x dim) of an empty sequence.  Returns their queries (q: tokens x query heads x dim), turned
        if the cache turns its keys."""
        if self.lengths[sequence]:
            raise ValueError("PagedCache.prefill: sequence %d holds %d tokens" % (sequence, self.lengths[sequence]))
        self._check_positions("prefill", positions)
        tokens, page = k.shape[0], self.page
        self._open([sequence], tokens)
        t = torch.arange(tokens, device=k.device)
        slots = self.table[sequence][t // page] * page + t % page
        q = self._store(q, k, v, slots.to(torch.int32), t, positions)
        full = tokens // page
        if full:
            self._keep_means(self.table[sequence, :full].long(),
                             k[:full * page].reshape(full, page, *k.shape[1:]) if self.frequencies is None else None)
        self.length[sequence] = self.lengths[sequence] = tokens
        return q

    def release(self, sequence):
        """Gives the pages of a sequence back."""
        self.free += self.held[sequence][::-1]
        self.held[sequence] = []
        self.length[sequence] = self.lengths[sequence] = 0

    def _append(self, q, k, v, positions):
        """A token more of every sequence.  Returns q as it is used and the lengths that the caller makes the cache's own when all is
        done: what was written counts from then on."""
        page, sequences = self.page, len(self.lengths)
        self._open(range(sequences), 1)
        at = self.table.gather(1, (self.length // page).long()[:, None])[:, 0]
        q = self._store(q, k, v, at * page + self.length % page, self.length, positions)
        length, lengths = self.length + 1, [n + 1 for n in self.lengths]
        if any(n % page == 0 for n in lengths):  # pages that are full now
            self._keep_means(torch.tensor([self.held[s][n // page - 1] for s, n in enumerate(lengths) if n % page == 0], device=k.device))
        return q, length, lengths

    def step(self, q, k, v, count, sink=1, local=2, scale=None, positions=None):
        """One token more of every sequence (k, v: sequences x heads x dim), and what it reads (q: sequences x query heads x
        dim) from the ``count`` best pages of each sequence and key-value head; the last ``local`` (at least 1) and first
        ``sink`` pages are always among them.  A sequence that was released begins anew with its token.  Where the call raises, the
        cache holds what it held before."""
        if local < 1:
            raise ValueError("PagedCache.step: the page of the token itself is always attended to: local = %d" % local)
        if sink < 0 or count < sink + local:
            raise ValueError("PagedCache.step: %d pages, the first %d and the last %d always among them" % (count, sink, local))
        self._check_positions("step", positions)
        page, sequences, groups = self.page, len(self.lengths), self.k.shape[1]
        if self.frequencies is None:
            q_codes, _ = _means(q[:, None], 1, groups)
        q, length, lengths = self._append(q, k, v, positions)
        if self.frequencies is not None:
            q_codes, _ = _means(q[:, None], 1, groups)

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

    def step_window(self, q, k, v, window, sink=0, scale=None, positions=None):
        """As ``step``, but a token reads the last ``window`` tokens of its sequence, itself among them, and the first ``sink``.  Pages that
        the window has left behind stay the sequence's until ``release``: another call may ask for more of them."""
        self._check_positions("step_window", positions)
        q, length, lengths = self._append(q, k, v, positions)
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        hip.paged_window_attention(q, self.k, self.v, self.table, length, out, window, sink, None, scale, self.k_scale, self.v_scale)
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
