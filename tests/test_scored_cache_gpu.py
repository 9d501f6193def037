"""Attention that adds up the weight of every cached key, the choice of the keys that stay and the moves that close the gaps,
each against its definition in 64 bits on the CPU: lengths from none to thousands, heads and pages of odd sizes, pools of NaN,
masked places that hold no numbers, scores with ties, infinities and NaN.

The bounds are derived, not fitted.  A score is a sum of D products in 32 bits: its error is taken as 4 sqrt(D) units of 2^-24 of
the sum of the products' magnitudes (a random walk with room), that of a capped one as eight units of the cap more.  A weight's
relative error is then twice that, and sums of up to L terms add sqrt(L) units; the exponential and the division 2^-20; weights
below 2^-126, the smallest 32-bit number that is not flushed, may be none.  In bfloat16
the weights are rounded to 8 bits for the second product and the output once more, each by up to 2^-8 of what is rounded."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F64 = torch.float64
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    from nanohybrid_vlm_b200.kernels import ops
    return ops


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Case:
    """Requests with ``news`` new tokens among ``lens`` keys over pages in no order, in a pool that starts as NaN."""

    def __init__(self, news, lens, nq, nkv, d, page, dtype, cap=None, sinks=False, seed=0, spread=1.5, width=0):
        g = torch.Generator().manual_seed(seed)
        self.news, self.lens, self.nq, self.nkv, self.d, self.page, self.dtype, self.cap = news, lens, nq, nkv, d, page, dtype, cap
        counts = [-(-L // page) for L in lens]
        self.n_pages = sum(counts) + 3
        ids = torch.randperm(self.n_pages, generator=g).tolist()
        self.table = torch.full((len(lens), max(counts + [1]) + width), -1, dtype=torch.int32)
        self.pages = torch.full((self.n_pages, 2, nkv, page, d), math.nan, dtype=dtype)
        self.scores = torch.full((self.n_pages, nkv, page), math.nan)
        self.births = torch.full((self.n_pages, nkv, page), -7, dtype=torch.int32)
        self.scale = d ** -0.5
        T = sum(news)
        self.q = (torch.randn(T, nq * d, generator=g) * spread).to(dtype)
        self.sinks = torch.randn(nq, generator=g) if sinks else None
        self.cu = [0]
        self.positions = []
        for s, (n, L) in enumerate(zip(news, lens)):
            self.table[s, :counts[s]] = torch.tensor([ids.pop() for _ in range(counts[s])], dtype=torch.int32)
            self.cu.append(self.cu[-1] + n)
            self.positions += [1000 * s + L - n + t for t in range(n)]
            for j in range(L):
                p, o = int(self.table[s, j // page]), j % page
                self.pages[p, :, :, o] = torch.randn(2, nkv, d, generator=g).to(dtype)
                self.scores[p, :, o] = torch.rand(nkv, generator=g) * 3
                self.births[p, :, o] = j
                if j >= L - n:
                    self.scores[p, :, o] = math.nan         # a new key has none yet
        self.lens_t, self.cu_t = i32(lens), i32(self.cu)

    def keys(self, s, g, plane):
        L = self.lens[s]
        rows = [self.pages[int(self.table[s, j // self.page]), plane, g, j % self.page] for j in range(L)]
        return torch.stack(rows).to(F64) if rows else torch.zeros(0, self.d, dtype=F64)

    def of(self, per_page, s, g):
        return torch.stack([per_page[int(self.table[s, j // self.page]), g, j % self.page] for j in range(self.lens[s])]) \
            if self.lens[s] else torch.zeros(0)

    def want(self):
        """(output, per request [nkv, L] the new weights, bounds of both) in 64 bits."""
        G = self.nq // self.nkv
        out, out_tol = torch.zeros(self.q.shape, dtype=F64), torch.zeros(self.q.shape, dtype=F64)
        weights, tols = [], []
        for s, (n, L) in enumerate(zip(self.news, self.lens)):
            w_s, t_s = torch.zeros(self.nkv, L, dtype=F64), torch.zeros(self.nkv, L, dtype=F64)
            for g in range(self.nkv):
                k, v = self.keys(s, g, 0), self.keys(s, g, 1)
                for h in range(g * G, (g + 1) * G):
                    rows = slice(self.cu[s], self.cu[s] + n)
                    x = self.q[rows, h * self.d:(h + 1) * self.d].to(F64)
                    z = x @ k.T * self.scale
                    err = (x.abs() @ k.abs().T * self.scale).amax() * 4 * math.sqrt(self.d) * 2 ** -24 if n and L else 0.0
                    if self.cap:
                        z = self.cap * torch.tanh(z / self.cap)
                        err += 8 * self.cap * 2 ** -24
                    for t in range(n):
                        z[t, L - n + t + 1:] = -torch.inf
                    norm = torch.logsumexp(z, 1, keepdim=True)
                    if self.sinks is not None:
                        norm = torch.logaddexp(norm, self.sinks[h].to(F64))
                    p = torch.exp(z - norm)
                    rel = 2 * err + math.sqrt(max(L, n * G)) * 2 ** -24 + 2 ** -20
                    out[rows, h * self.d:(h + 1) * self.d] = p @ v
                    # the weights' error times the values they weigh, and what is rounded to 8 bits
                    unit = 2 * 2 ** -8 if self.dtype == torch.bfloat16 else 0.0
                    out_tol[rows, h * self.d:(h + 1) * self.d] = (p @ v.abs()) * (rel + unit) + 2 ** -20 * (p @ v.abs())
                    w_s[g] += p.sum(0)
                    t_s[g] += p.sum(0) * rel + n * 2.0 ** -126      # a weight below the smallest 32-bit number is none
            weights.append(w_s)
            tols.append(t_s)
        return out, out_tol, weights, tols

    def run(self, ops, in_place=False, q=None, births=True, table=None):
        dev = dict(q=(self.q if q is None else q).cuda(), pages=self.pages.cuda(), scores=self.scores.cuda(), births=self.births.cuda(),
                   table=(self.table if table is None else table).cuda())
        out = torch.full_like(dev["q"], math.nan)
        scores_out = dev["scores"] if in_place else torch.full_like(dev["scores"], 5.0)
        ops.attention_scored(out, dev["q"], dev["pages"], dev["scores"], dev["table"], self.cu_t, self.lens_t, len(self.lens),
                             min(self.news), max(self.news), max(self.lens), self.nq, self.nkv, self.d, self.scale,
                             births=dev["births"] if births else None, positions=i32(self.positions) if births else None,
                             sinks=None if self.sinks is None else self.sinks.cuda(), softcap=self.cap,
                             scores_out=None if in_place else scores_out)
        torch.cuda.synchronize()
        ops.raise_wait_errors()
        return out.cpu(), scores_out.cpu(), dev["births"].cpu()

    def check(self, out, scores_out, births=None, rows=None):
        want, tol, weights, tols = self.want()
        err = (out.to(F64) - want).abs()
        rows = slice(None) if rows is None else rows
        assert not torch.isnan(out[rows].float()).any()
        assert (err <= tol)[rows].all(), (err / tol.clamp(min=1e-30))[rows].max()
        touched = torch.zeros_like(self.scores, dtype=torch.bool)
        for s, (n, L) in enumerate(zip(self.news, self.lens)):
            for g in range(self.nkv):
                old = self.of(self.scores, s, g).to(F64)
                old[L - n:] = 0
                got = self.of(scores_out, s, g).to(F64)
                bound = tols[s][g] + (old + weights[s][g]) * 2 ** -22
                diff = (got - old - weights[s][g]).abs()
                assert (diff <= bound).all(), (s, g, (diff / bound.clamp(min=1e-30)).max())
            for j in range(L):
                touched[int(self.table[s, j // self.page]), :, j % self.page] = True
        if births is not None:
            expect = self.births.clone()
            for s, (n, L) in enumerate(zip(self.news, self.lens)):
                for t in range(n):
                    j = L - n + t
                    expect[int(self.table[s, j // self.page]), :, j % self.page] = self.positions[self.cu[s] + t]
            assert torch.equal(births, expect)
        return touched


SHAPES = [(4, 2, 16, 16), (6, 2, 32, 8), (8, 8, 64, 64), (12, 4, 64, 16), (16, 2, 128, 256), (8, 2, 128, 32), (6, 1, 96, 24), (5, 1, 80, 7),
          (3, 3, 256, 64), (40, 2, 64, 64), (2, 1, 33, 5), (7, 7, 8, 1), (4, 4, 192, 64), (64, 1, 128, 64)]
LENGTHS = {
    "single": ([1, 1, 1, 1], [1, 2, 65, 300]),
    "prompts": ([70, 1, 33, 129], [70, 40, 97, 300]),
    "few": ([3, 5, 0, 2], [200, 5, 17, 131]),
    "one": ([1], [1]),
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page", SHAPES)
@pytest.mark.parametrize("lengths", LENGTHS)
def test_outputs_weights_and_births(ops, dtype, nq, nkv, d, page, lengths):
    c = Case(*LENGTHS[lengths], nq, nkv, d, page, dtype, seed=nq * d + page)
    out, scores_out, births = c.run(ops)
    touched = c.check(out, scores_out, births)
    assert (scores_out[~touched] == 5.0).all()              # slots of no request stay as they are


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page", [(8, 2, 128, 64), (6, 2, 32, 8), (12, 4, 64, 16)])
@pytest.mark.parametrize("cap,sinks,spread", [(30.0, False, 1.5), (2.0, True, 20.0), (None, True, 1.5), (50.0, True, 60.0)])
def test_caps_and_sinks(ops, dtype, nq, nkv, d, page, cap, sinks, spread):
    for lengths in ("single", "prompts", "few"):
        c = Case(*LENGTHS[lengths], nq, nkv, d, page, dtype, cap=cap, sinks=sinks, spread=spread, seed=3)
        c.check(*c.run(ops))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page,news,lens", [
    (8, 2, 128, 256, [1, 1], [5000, 3]),                    # one long request beside a short one
    (8, 1, 64, 64, [1], [9001]),
    (4, 1, 128, 64, [700], [700]),
    (2, 1, 128, 64, [300, 40], [2900, 40]),
    (4, 4, 64, 32, [17, 1, 600], [4000, 2000, 601]),
    (16, 2, 128, 64, [4, 9, 2], [3000, 700, 2]),
    (16, 1, 64, 8, [130] * 3, [130, 1000, 260]),
])
def test_long_requests(ops, dtype, nq, nkv, d, page, news, lens):
    c = Case(news, lens, nq, nkv, d, page, dtype, seed=len(lens) + page)
    c.check(*c.run(ops))


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_requests(ops, dtype):
    lens = [1 + (37 * i) % 90 for i in range(150)]
    c = Case([1 + i % 3 if lens[i] > 3 else 1 for i in range(150)], lens, 4, 2, 64, 64, dtype, seed=8)
    c.check(*c.run(ops))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page,new,cap,sinks", [
    (4, 1, 128, 64, 1, None, True),
    (8, 1, 128, 16, 2, 30.0, False),
    (3, 3, 40, 7, 2, 5.0, True),
    (8, 8, 64, 8, 1, None, False),
    (16, 1, 32, 48, 1, 20.0, True),
    (2, 1, 256, 32, 1, None, True),
])
def test_more_blocks_than_run_at_once(ops, dtype, nq, nkv, d, page, new, cap, sinks):
    """Few rows a request, of so many requests that parts and weights are brought together by a kernel of their own; some bring nothing."""
    lens = [3 + (53 * i) % 127 for i in range(120)]
    c = Case([(new * (i % 5 > 0)) for i in range(120)], lens, nq, nkv, d, page, dtype, cap=cap, sinks=sinks, seed=12)
    c.check(*c.run(ops))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths", ["single", "prompts"])
def test_in_place_rows_apart_and_a_wide_table(ops, dtype, lengths):
    c = Case(*LENGTHS[lengths], 8, 2, 64, 64, dtype, seed=5, width=3)
    T = c.q.shape[0]
    wide = torch.full((T, 8 * 64 + 64), math.nan, dtype=dtype)
    wide[:, :8 * 64] = c.q
    q = wide.cuda()[:, :8 * 64]
    out = torch.full((T, 8 * 64 + 32), 9.0, dtype=dtype, device="cuda")
    scores, births, pages = c.scores.cuda(), c.births.cuda(), c.pages.cuda()
    table = torch.full((len(c.lens), c.table.shape[1] + 5), 12345, dtype=torch.int32)
    table[:, :c.table.shape[1]] = c.table
    ops.attention_scored(out[:, :8 * 64], q, pages, scores, table.cuda()[:, :c.table.shape[1]], c.cu_t, c.lens_t, len(c.lens), min(c.news),
                         max(c.news), max(c.lens), 8, 2, 64, c.scale, births=births, positions=i32(c.positions))
    c.check(out[:, :8 * 64].cpu(), scores.cpu(), births.cpu())
    assert (out[:, 8 * 64:] == 9.0).all()
    again, scores_again, _ = c.run(ops, births=False)       # without births, and out of place: the same numbers
    assert torch.equal(out[:, :8 * 64].cpu(), again)
    L = c.lens[-1]
    assert torch.equal(c.of(scores.cpu(), len(c.lens) - 1, 1)[:L], c.of(scores_again, len(c.lens) - 1, 1)[:L])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,page", [(128, 64), (32, 8), (64, 256)])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_what_a_token_does_not_see_does_not_reach_it(ops, dtype, d, page, what):
    """Key or value of the token in the middle of a portion is no number: earlier tokens do not notice, and later ones of a
    request of their own neither."""
    n = 80
    c = Case([n, 1, 50], [n + 40, 30, 50], 4, 2, d, page, dtype, seed=d)
    clean, scores_clean, _ = c.run(ops)
    bad = 40 + 45                                           # the slot of the first request's 46th new token
    for plane in (0, 1):
        pages = c.pages.clone()
        c.pages[int(c.table[0, bad // page]), plane, :, bad % page] = what
        out, scores_out, _ = c.run(ops)
        c.pages = pages
        assert torch.equal(out[:45], clean[:45]) and torch.equal(out[n:], clean[n:])
        if plane == 1:
            assert not torch.isfinite(out[45:n].float()).any()          # p v of a value that is no number, for every later token
            for s in range(3):                                          # weights do not depend on values
                assert torch.equal(c.of(scores_out, s, 0), c.of(scores_clean, s, 0))
        for s in (1, 2):
            assert torch.equal(c.of(scores_out, s, 1), c.of(scores_clean, s, 1))


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_any_size(ops, dtype):
    """Products that reach the ends of the exponential: one key takes all, or all keys tie."""
    c = Case([9, 1], [90, 70], 4, 2, 64, 64, dtype, seed=2, spread=300.0)
    c.check(*c.run(ops))
    c = Case([9, 1], [90, 70], 4, 2, 64, 64, dtype, seed=2, spread=0.0)
    out, scores_out, births = c.run(ops)
    c.check(out, scores_out, births)
    c = Case([9, 1], [90, 70], 4, 2, 64, 64, dtype, seed=2, spread=1e-30)
    c.check(*c.run(ops))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths", ["single", "prompts", "few"])
def test_the_same_call_gives_the_same_bits_on_any_stream(ops, dtype, lengths):
    c = Case(*LENGTHS[lengths], 8, 2, 128, 64, dtype, seed=4)
    first = c.run(ops)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = c.run(ops)
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(first[:2], second[:2]))


def test_requests_without_keys_and_entries_without_pages(ops):
    for dtype in DTYPES:
        # an entry that only pads a batch: one token, no page
        c = Case([1, 1, 0], [30, 1, 0], 4, 2, 64, 64, dtype, seed=6)
        c.table[1] = -1
        out, scores_out, _ = c.run(ops)
        assert (out[1] == 0).all() and not torch.isnan(out.float()).any()
        c = Case([20, 0], [20, 45], 4, 2, 64, 64, dtype, seed=6)        # a request that brings nothing keeps its scores
        _, scores_out, _ = c.run(ops)
        assert torch.equal(c.of(scores_out, 1, 0), c.of(c.scores, 1, 0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 24])
def test_offsets_beyond_32_bits(ops, dtype, new):
    """The pages in use stand at the end of a pool of more than 2^32 elements, and half of them at its start."""
    c = Case([new, 1], [90, 70], 4, 2, 64, 64, dtype, seed=8)
    n_pages = 2 ** 32 // c.pages[0].numel() + 5
    shift = n_pages - c.n_pages
    where = torch.tensor([i if i % 2 else i + shift for i in range(c.n_pages)])
    pages = torch.empty(n_pages, *c.pages.shape[1:], dtype=dtype, device="cuda")
    scores, births = torch.empty(n_pages, 2, 64, device="cuda"), torch.empty(n_pages, 2, 64, dtype=torch.int32, device="cuda")
    pages[where], scores[where], births[where] = c.pages.cuda(), c.scores.cuda(), c.births.cuda()
    table = torch.where(c.table >= 0, where[c.table.long().clamp(min=0)].int(), c.table).cuda()
    out = torch.full_like(c.q, math.nan).cuda()
    ops.attention_scored(out, c.q.cuda(), pages, scores, table, c.cu_t, c.lens_t, 2, 1, new, 90, 4, 2, 64, c.scale, births=births,
                         positions=i32(c.positions))
    ops.raise_wait_errors()
    c.check(out.cpu(), scores[where].cpu(), births[where].cpu())
    before = pages[where].cpu()
    moves = torch.tensor([[[64, 66, 80]] * 2, [[65, 69, -1]] * 2], dtype=torch.int32), torch.tensor([[[3, 0, 63]] * 2, [[1, 2, -1]] * 2], dtype=torch.int32)
    ops.move_keys(pages, scores, births, table, moves[0].cuda(), moves[1].cuda(), 2)
    for s in range(2):
        for a, b in zip(moves[0][s, 0].tolist(), moves[1][s, 0].tolist()):
            if a >= 0:
                before[int(c.table[s, b // 64]), :, :, b % 64] = before[int(c.table[s, a // 64]), :, :, a % 64]
    assert torch.equal(pages[where].cpu().nan_to_num(7.0), before.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths_far_below_the_longest_allowed(ops, dtype):
    """The caller's bound on the lengths is what the scratch is sized by: beyond its largest size the requests go in groups."""
    c = Case([1, 2, 1, 2, 0], [90, 70, 1, 129, 20], 16, 2, 64, 64, dtype, seed=9)
    bound = 2 ** 21
    table = torch.full((5, bound // 64), -1, dtype=torch.int32)
    table[:, :c.table.shape[1]] = c.table
    scores, births, out = c.scores.cuda(), c.births.cuda(), torch.full_like(c.q, math.nan).cuda()
    ops.attention_scored(out, c.q.cuda(), c.pages.cuda(), scores, table.cuda(), c.cu_t, c.lens_t, 5, 0, 2, bound, 16, 2, 64, c.scale,
                         births=births, positions=i32(c.positions))
    ops.raise_wait_errors()
    c.check(out.cpu(), scores.cpu(), births.cpu())


def test_refusals_of_attention(ops):
    from nanohybrid_vlm_b200.kernels.library import KernelError
    c = Case([2, 1], [40, 30], 4, 2, 64, 16, torch.bfloat16)
    base = dict(out=torch.empty_like(c.q).cuda(), q=c.q.cuda(), kv_pages=c.pages.cuda(), scores=c.scores.cuda(), block_table=c.table.cuda(),
                cu_q=c.cu_t, kv_len=c.lens_t, n_seqs=2, min_new=1, max_new=2, max_kv_len=40, nq=4, nkv=2, head_dim=64, scale=0.125)
    ops.attention_scored(**base)
    wrong = [dict(q=c.q), dict(q=c.q.float().cuda()), dict(nq=3), dict(nkv=4), dict(head_dim=32), dict(scores=c.scores.cuda()[:, :1]),
             dict(scores=c.scores.cuda().half()), dict(scores=c.scores.cuda()[:-1]), dict(block_table=c.table.cuda().long()),
             dict(block_table=c.table.cuda()[:1]), dict(max_kv_len=100000), dict(cu_q=c.cu_t[:2]), dict(kv_len=c.lens_t.long()), dict(min_new=3),
             dict(max_new=1), dict(births=c.births.cuda()), dict(positions=i32(c.positions)), dict(births=c.births.cuda(), positions=i32([1])),
             dict(births=c.births.cuda().float(), positions=i32(c.positions)), dict(sinks=torch.zeros(3).cuda()), dict(softcap=-1.0), dict(softcap=0.0),
             dict(scores_out=c.scores.cuda()[1:]), dict(out=torch.empty(3, 8).cuda()), dict(kv_pages=c.pages.cuda().transpose(2, 3)),
             dict(kv_pages=c.pages.cuda().half(), q=c.q.cuda().half(), out=c.q.cuda().half())]
    for change in wrong:
        with pytest.raises(KernelError):
            ops.attention_scored(**{**base, **change})
    big = Case([1], [3], 1, 1, 257, 4, torch.float32)
    with pytest.raises(KernelError):
        big.run(ops)


# ---------------------------------------------------------------- which keys stay
def choose(scores, births, lens, seen, budgets, keep_first, keep_recent):
    """The definition, slot by slot: per request and head the moves (source, target) in order."""
    out = []
    for s, L in enumerate(lens):
        per_head = []
        for g in range(scores[s].shape[0]):
            def value(j):
                b, x = int(births[s][g, j]), float(scores[s][g, j])
                if b < keep_first or b >= seen[s] - keep_recent:
                    return math.inf
                return x
            vals = [value(j) for j in range(L)]
            order = sorted(range(L), key=lambda j: (math.isnan(vals[j]), -vals[j] if not math.isnan(vals[j]) else 0.0, j))
            kept = set(order[:max(0, budgets[s])])
            sources = [j for j in range(L) if j in kept and j >= budgets[s]]
            targets = [j for j in range(L) if j not in kept and j < budgets[s]]
            per_head.append(list(zip(sources, targets)))
        out.append(per_head)
    return out


class Pool:
    def __init__(self, lens, nkv, page, seed=0, d=0, dtype=torch.float32):
        g = torch.Generator().manual_seed(seed)
        counts = [-(-L // page) for L in lens]
        n_pages = sum(counts) + 2
        ids = torch.randperm(n_pages, generator=g).tolist()
        self.lens, self.nkv, self.page, self.n_pages = lens, nkv, page, n_pages
        self.table = torch.full((len(lens), max(counts + [1])), -1, dtype=torch.int32)
        for s, c in enumerate(counts):
            self.table[s, :c] = torch.tensor([ids.pop() for _ in range(c)], dtype=torch.int32)
        self.scores = torch.full((n_pages, nkv, page), math.nan)
        self.births = torch.full((n_pages, nkv, page), -1, dtype=torch.int32)
        if d:
            self.pages = torch.randn(n_pages, 2, nkv, page, d, generator=g).to(dtype)
        self.gen = g

    def fill(self, scores, births):
        """Lists per request of [nkv, L]."""
        for s, L in enumerate(self.lens):
            for p in range(-(-L // self.page)):
                a, b = p * self.page, min(L, (p + 1) * self.page)
                self.scores[int(self.table[s, p]), :, :b - a] = scores[s][:, a:b]
                self.births[int(self.table[s, p]), :, :b - a] = births[s][:, a:b]

    def random(self, ties, order=True):
        scores, births = [], []
        for L in self.lens:
            x = torch.randn(self.nkv, L, generator=self.gen).exp()
            scores.append((x * 4).round() / 4 if ties else x)
            b = torch.stack([torch.randperm(2 * L + 1, generator=self.gen)[:L] for _ in range(self.nkv)]) if L else torch.zeros(self.nkv, 0)
            births.append((b.sort(1).values if order else b).int())
        self.fill(scores, births)
        return scores, births

    def select(self, ops, seen, budgets, keep_first, keep_recent, room=None):
        M = max([0] + [min(max(0, b), max(0, L - b)) for L, b in zip(self.lens, budgets)]) if room is None else room
        sources = torch.full((len(self.lens), self.nkv, M), 99, dtype=torch.int32, device="cuda")
        targets = torch.full_like(sources, 99)
        ops.select_keys(sources, targets, self.scores.cuda(), self.births.cuda(), self.table.cuda(), i32(self.lens), i32(seen), i32(budgets),
                        len(self.lens), max(self.lens), keep_first, keep_recent)
        return sources, targets

    def check(self, ops, scores, births, seen, budgets, keep_first, keep_recent, room=None):
        sources, targets = self.select(ops, seen, budgets, keep_first, keep_recent, room)
        ops.raise_wait_errors()
        want = choose(scores, births, self.lens, seen, budgets, keep_first, keep_recent)
        for s in range(len(self.lens)):
            for g in range(self.nkv):
                got = list(zip(sources[s, g].tolist(), targets[s, g].tolist()))
                n = len(want[s][g])
                assert got[:n] == want[s][g] and all(x == (-1, -1) for x in got[n:]), (s, g)
        return sources, targets


@pytest.mark.parametrize("nkv,page,lens,budgets", [
    (2, 16, [100, 31, 64, 1, 0], [40, 31, 1, 1, 5]),
    (1, 1, [57], [20]),
    (3, 7, [2000, 1999, 600], [600, 1, 599]),
    (8, 256, [2304, 2049, 700, 2304], [2048, 2048, 2048, 0]),
    (1, 64, [9000], [4500]),
    (2, 256, [40001, 12], [4096, 4096]),
    (4, 32, [600], [599]),
    (1, 16, [70000], [69000]),
])
@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("keep_first,keep_recent", [(0, 0), (4, 9), (3, 100000)])
def test_the_keys_that_stay(ops, nkv, page, lens, budgets, ties, keep_first, keep_recent):
    p = Pool(lens, nkv, page, seed=page + len(lens))
    scores, births = p.random(ties, order=page != 32)
    p.check(ops, scores, births, [2 * L + 1 for L in lens], budgets, keep_first, keep_recent)


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("budget", [4096, 330000])
def test_more_keys_than_the_blocks_hold(ops, ties, budget):
    """Beyond what the blocks of a cluster keep in shared memory the keys are read again in each pass."""
    p = Pool([350000, 400], 1, 256, seed=11)
    scores, births = p.random(ties)
    p.check(ops, scores, births, [700001, 801], [budget, 300], 4, 512)


def test_scores_that_are_alike_infinite_or_no_numbers(ops):
    L = 300
    p = Pool([L, L, L, L], 2, 16, seed=1)
    scores, births = p.random(False)
    odd = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1e-45, 3.4e38, -3.4e38, 1.0])
    scores[0] = odd.repeat(2, L // 10)
    scores[1] = torch.full((2, L), 2.5)
    scores[2] = torch.full((2, L), math.nan)
    scores[3] = torch.where(torch.arange(L) % 2 == 0, 0.0, -0.0).repeat(2, 1)
    p.fill(scores, births)
    for budget in (1, 29, 30, 31, 150, 299):
        p.check(ops, scores, births, [2 * L + 1] * 4, [budget] * 4, 0, 0)
    p.check(ops, scores, births, [2 * L + 1] * 4, [150] * 4, 7, 30)


def test_room_for_moves(ops):
    from nanohybrid_vlm_b200.kernels.library import KernelError
    p = Pool([64], 1, 16, seed=2)
    scores = [torch.arange(64).float().view(1, -1)]
    births = [torch.arange(64, dtype=torch.int32).view(1, -1)]
    p.fill(scores, births)
    p.check(ops, scores, births, [64], [20], 0, 0, room=20)
    p.check(ops, scores, births, [64], [20], 0, 0, room=50)
    p.select(ops, [64], [20], 0, 0, room=19)                # one too few: the next check of the kernels says so
    with pytest.raises(KernelError, match="key_eviction"):
        ops.raise_wait_errors()
    ops.raise_wait_errors()


def test_refusals_of_the_choice_and_the_moves(ops):
    from nanohybrid_vlm_b200.kernels.library import KernelError
    p = Pool([40], 2, 16, seed=3, d=8)
    p.random(False)
    moves = torch.full((1, 2, 20), -1, dtype=torch.int32, device="cuda")
    base = dict(sources=moves, targets=moves.clone(), scores=p.scores.cuda(), births=p.births.cuda(), block_table=p.table.cuda(), kv_len=i32([40]),
                seen=i32([40]), budgets=i32([20]), n_seqs=1, max_kv_len=40, keep_first=0, keep_recent=0)
    ops.select_keys(**base)
    for change in (dict(sources=moves[:, :1]), dict(targets=moves[..., :10].contiguous()), dict(sources=moves.long()), dict(scores=p.scores),
                   dict(births=None), dict(births=p.births.cuda().long()), dict(kv_len=i32([])), dict(seen=torch.zeros(1).cuda()), dict(budgets=i32([])),
                   dict(max_kv_len=1000), dict(keep_first=-1), dict(keep_recent=-1), dict(block_table=p.table.cuda().long())):
        with pytest.raises(KernelError):
            ops.select_keys(**{**base, **change})
    base = dict(kv_pages=p.pages.cuda(), scores=p.scores.cuda(), births=p.births.cuda(), block_table=p.table.cuda(), sources=moves, targets=moves, n_seqs=1)
    ops.move_keys(**base)
    for change in (dict(kv_pages=p.pages), dict(kv_pages=p.pages.cuda().half()), dict(kv_pages=p.pages.cuda()[:-1]), dict(births=None),
                   dict(sources=moves[:, :1]), dict(n_seqs=2), dict(scores=p.scores.cuda().double())):
        with pytest.raises(KernelError):
            ops.move_keys(**{**base, **change})


# ---------------------------------------------------------------- the moves
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nkv,d,page,lens,budgets", [
    (2, 64, 16, [100, 31, 64, 0], [40, 31, 1, 5]),
    (1, 33, 7, [500], [200]),
    (8, 128, 256, [2304, 700], [2048, 600]),
    (3, 8, 64, [1000], [10]),
    (2, 256, 32, [90], [45]),
    (1, 1, 1, [20], [7]),
])
def test_the_moves(ops, dtype, nkv, d, page, lens, budgets):
    p = Pool(lens, nkv, page, seed=d, d=d, dtype=dtype)
    scores, births = p.random(False)
    sources, targets = p.select(ops, [2 * L + 1 for L in lens], budgets, 2, 5)
    pages, sc, bi = p.pages.cuda(), p.scores.cuda(), p.births.cuda()
    for _ in range(2):                                      # twice is the same as once
        ops.move_keys(pages, sc, bi, p.table.cuda(), sources, targets, len(lens))
    want_pages, want_sc, want_bi = p.pages.clone(), p.scores.clone(), p.births.clone()
    for s in range(len(lens)):
        for g in range(nkv):
            for a, b in zip(sources[s, g].tolist(), targets[s, g].tolist()):
                if a < 0:
                    continue
                pa, pb = int(p.table[s, a // page]), int(p.table[s, b // page])
                want_pages[pb, :, g, b % page] = p.pages[pa, :, g, a % page]
                want_sc[pb, g, b % page] = p.scores[pa, g, a % page]
                want_bi[pb, g, b % page] = p.births[pa, g, a % page]
    assert torch.equal(pages.cpu(), want_pages) and torch.equal(bi.cpu(), want_bi)
    assert torch.equal(sc.cpu().nan_to_num(-1.0), want_sc.nan_to_num(-1.0))
    # what stays are the largest scores, whatever order they lie in
    for s, (L, b) in enumerate(zip(lens, budgets)):
        at = [(int(p.table[s, j // page]), j % page) for j in range(min(L, b))]
        for g in range(nkv):
            kept = sorted(int(bi[q, g, o]) for q, o in at)
            held = [(int(births[s][g, j]), float(scores[s][g, j])) for j in range(L)]
            held = [(math.inf if t < 2 or t >= 2 * L + 1 - 5 else x, t) for t, x in held]
            assert kept == sorted(t for _, t in sorted(held, key=lambda v: -v[0])[:b])


def test_moves_beyond_the_table_move_nothing(ops):
    p = Pool([40], 1, 16, seed=3, d=8)
    p.random(False)
    bad = torch.tensor([[[1000, 5, -1, 39]]], dtype=torch.int32, device="cuda")
    to = torch.tensor([[[1, 4000, 3, -1]]], dtype=torch.int32, device="cuda")
    pages, sc, bi = p.pages.cuda(), p.scores.cuda(), p.births.cuda()
    ops.move_keys(pages, sc, bi, p.table.cuda(), bad, to, 1)
    assert torch.equal(pages.cpu(), p.pages) and torch.equal(bi.cpu(), p.births)


# ---------------------------------------------------------------- steps that bring nothing
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page", [(4, 2, 64, 16), (64, 1, 128, 64), (3, 3, 33, 5), (2, 1, 256, 7)])
@pytest.mark.parametrize("lens", [[40, 0, 7], [20000], [3 + i % 90 for i in range(130)]])
def test_a_step_without_new_tokens_passes_the_scores_through(ops, dtype, nq, nkv, d, page, lens):
    c = Case([0] * len(lens), [min(L, 90) for L in lens], nq, nkv, d, page, dtype, seed=13)
    scores_out = torch.full_like(c.scores, 5.0).cuda()
    q = torch.empty(0, nq * d, dtype=dtype, device="cuda")
    births = c.births.cuda()
    longest = max(lens)
    table = torch.full((len(lens), -(-longest // page)), -1, dtype=torch.int32)
    table[:, :c.table.shape[1]] = c.table[:, :table.shape[1]]
    ops.attention_scored(torch.empty_like(q), q, c.pages.cuda(), c.scores.cuda(), table.cuda(), c.cu_t, c.lens_t, len(lens), 0, 0, longest, nq, nkv, d,
                         c.scale, births=births, positions=i32([]), scores_out=scores_out)
    ops.raise_wait_errors()
    touched = c.check(c.q, scores_out.cpu(), births.cpu(), rows=slice(0))
    assert (scores_out.cpu()[~touched] == 5.0).all()
    for s in range(len(lens)):
        for g in range(nkv):
            assert torch.equal(c.of(scores_out.cpu(), s, g), c.of(c.scores, s, g))


# ---------------------------------------------------------------- numbers that are none, and infinite ones, in sight
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page", [(4, 2, 128, 64), (6, 2, 32, 8), (2, 2, 64, 256), (3, 1, 33, 7)])
@pytest.mark.parametrize("cap,spread", [(None, 1.5), (30.0, 1.5), (30.0, 60.0), (2.0, 20.0)])
def test_scores_that_are_no_numbers_stay_so_under_a_cap(ops, dtype, nq, nkv, d, page, cap, spread):
    """The key of the 46th new token is no number: nobody before it notices, and from it on nothing is a number, whether the tile's other
    scores are small or beyond half the cap.  The same for a query, alone among its request's."""
    n, G = 80, nq // nkv
    c = Case([n, 1, 50, 3], [n + 40, 30, 50, 90], nq, nkv, d, page, dtype, cap=cap, spread=spread, seed=d)
    clean, scores_clean, _ = c.run(ops)
    bad, pages = 40 + 45, c.pages.clone()
    c.pages[int(c.table[0, bad // page]), 0, :, bad % page] = math.nan
    c.pages[int(c.table[1, 20 // page]), 0, :, 20 % page, d // 2] = math.nan           # an old key of a single token
    out, scores_out, _ = c.run(ops)
    c.pages = pages
    assert torch.equal(out[:45], clean[:45]) and torch.equal(out[n + 1:], clean[n + 1:])
    assert torch.isnan(out[45:n + 1].float()).all()
    for g in range(nkv):
        assert torch.isnan(c.of(scores_out, 0, g)).all() and torch.isnan(c.of(scores_out, 1, g)).all()
        for s in (2, 3):
            assert torch.equal(c.of(scores_out, s, g), c.of(scores_clean, s, g))
    q = c.q.clone()
    rows = [7, n, n + 1 + 20, n + 1 + 50 + 1]               # a token of each request, with its first head of the last KV head
    head = (nkv - 1) * G
    for r in rows:
        q[r, head * d] = math.nan
    out, scores_out, _ = c.run(ops, q=q)
    for t in range(q.shape[0]):
        got, want = out[t].view(nq, d), clean[t].view(nq, d)
        if t in rows:
            assert torch.isnan(got[head].float()).all()
            got, want = torch.cat([got[:head], got[head + 1:]]), torch.cat([want[:head], want[head + 1:]])
        assert torch.equal(got, want)
    for s, (r, L, new) in enumerate(zip((7, 0, 20, 1), c.lens, c.news)):
        assert torch.isnan(c.of(scores_out, s, nkv - 1)[:L - new + r + 1]).all()           # every key that the query sees


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page", [(6, 2, 64, 64), (5, 1, 128, 16), (4, 1, 128, 64), (7, 7, 40, 8)])
@pytest.mark.parametrize("news,lens", [([200, 3, 1], [700, 300, 65]), ([1, 2], [40, 90])])
def test_keys_of_minus_infinity_weigh_nothing(ops, dtype, nq, nkv, d, page, news, lens):
    """A key that every query's product with is minus infinity is a key of no weight, as one of -1e30 is."""
    c = Case(news, lens, nq, nkv, d, page, dtype, seed=17)
    c.q.view(-1, nq, d)[:, :, 3] = c.q.view(-1, nq, d)[:, :, 3].abs() + 0.5
    got = []
    for value in (-1e30, -math.inf):
        for s, L in enumerate(lens):
            for j in (5, L // 2, L - news[s]):              # the last one is the first new token's own
                c.pages[int(c.table[s, j // page]), 0, :, j % page, 3] = value
        got.append(c.run(ops))
    assert not torch.isnan(got[0][0].float()).any()
    assert torch.equal(got[0][0], got[1][0])
    for s in range(len(lens)):
        for g in range(nkv):
            assert torch.equal(c.of(got[0][1], s, g), c.of(got[1][1], s, g))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page,n", [(4, 2, 128, 64, 8), (2, 2, 64, 8, 5), (20, 4, 96, 16, 6), (3, 1, 40, 24, 4), (2, 1, 256, 64, 4), (8, 1, 32, 256, 4)])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_values_of_later_tokens_do_not_reach_earlier_ones_among_few(ops, dtype, nq, nkv, d, page, n, what):
    """The same for drafts: few tokens of several requests, the value of each of them no number in turn."""
    c = Case([n, n, 1], [n + 150, n, 30], nq, nkv, d, page, dtype, seed=d)
    clean, scores_clean, _ = c.run(ops)
    for bad in range(n):
        pages = c.pages.clone()
        for s in (0, 1):
            j = c.lens[s] - n + bad
            c.pages[int(c.table[s, j // page]), 1, :, j % page] = what
        out, scores_out, _ = c.run(ops)
        c.pages = pages
        for s in (0, 1):
            assert torch.equal(out[s * n:s * n + bad], clean[s * n:s * n + bad])
            assert not torch.isfinite(out[s * n + bad:(s + 1) * n].float()).any()
        assert torch.equal(out[2 * n:], clean[2 * n:])
        for s in range(3):
            for g in range(nkv):
                assert torch.equal(c.of(scores_out, s, g), c.of(scores_clean, s, g))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page", [(4, 2, 128, 64), (2, 2, 64, 16), (20, 1, 32, 8), (12, 2, 96, 64), (2, 1, 256, 64)])
@pytest.mark.parametrize("lengths", ["single", "few", "prompts"])
@pytest.mark.parametrize("what", [math.inf, -math.inf])
def test_infinite_values_in_sight(ops, dtype, nq, nkv, d, page, lengths, what):
    """One element of a value is infinite: so is that element of every output that sees it, and nothing else changes."""
    c = Case(*LENGTHS[lengths], nq, nkv, d, page, dtype, seed=19, spread=0.5)
    clean, scores_clean, _ = c.run(ops)
    e, slots = d - 3, [L * 2 // 3 for L in c.lens]
    for s, j in enumerate(slots):
        c.pages[int(c.table[s, j // page]), 1, :, j % page, e] = what
    out, scores_out, _ = c.run(ops)
    for s, (n, L) in enumerate(zip(c.news, c.lens)):
        for t in range(n):
            got, want = out[c.cu[s] + t].view(nq, d), clean[c.cu[s] + t].view(nq, d).clone()
            if slots[s] <= L - n + t:
                want[:, e] = what
            assert torch.equal(got, want), (s, t)
        for g in range(nkv):
            assert torch.equal(c.of(scores_out, s, g), c.of(scores_clean, s, g))


@pytest.mark.parametrize("nq,nkv,d,page", [(6, 2, 32, 8), (4, 2, 64, 64), (5, 1, 128, 16), (3, 1, 192, 64)])
def test_capped_scores_do_not_depend_on_what_lies_about(ops, nq, nkv, d, page):
    """Unused slots of the request's pages, entries without a page, the next request's queries and what the launch before left in shared
    memory: none of it shows, not in the last bit either."""
    c = Case([80, 3, 50, 1], [117, 30, 350, 70], nq, nkv, d, page, torch.bfloat16, cap=30.0, seed=d)
    c.table[2, 1] = -1
    before = Case([300], [300], nq, nkv, d, page, torch.bfloat16, cap=30.0, seed=1)
    empty, results = torch.isnan(c.pages), []
    for fill in (0.0, 5000.0):
        c.pages[empty] = fill
        before.q = torch.full_like(before.q, fill)
        before.run(ops)
        q = c.q.clone()
        if fill:
            q[83:133] *= 100                                # the third request's, behind those of the first two in a tile
        results.append(c.run(ops, q=q))
    (out, scores, _), (out2, scores2, _) = results
    assert torch.equal(out[:83], out2[:83]) and torch.equal(out[133:], out2[133:])
    for s in (0, 1, 3):
        for g in range(nkv):
            assert torch.equal(c.of(scores, s, g), c.of(scores2, s, g))
    out3, scores3, _ = c.run(ops)
    assert torch.equal(out3, out)
    held = [j for j in range(350) if j // page != 1]
    assert torch.equal(c.of(scores3, 2, 0)[held], c.of(scores, 2, 0)[held])


@pytest.mark.parametrize("nq,nkv,d,page", [(4, 2, 128, 64), (6, 2, 64, 8), (1, 1, 32, 16), (8, 1, 256, 64)])
@pytest.mark.parametrize("first", [0, 70])
def test_odd_values_that_only_the_second_tile_of_a_block_sees(ops, nq, nkv, d, page, first):
    """A block's two tiles of rows end at unlike keys: what the later one finds in its own last keys is its own business."""
    n, old = 150, 90
    c = Case([n, 2], [n + old, 64], nq, nkv, d, page, torch.bfloat16, seed=d)
    clean, scores_clean, _ = c.run(ops)
    for bad in range(first, n, 13):
        pages = c.pages.clone()
        for j in range(old + bad, old + n, 29):
            c.pages[int(c.table[0, j // page]), 1, :, j % page] = math.nan if j % 2 else math.inf
        out, scores_out, _ = c.run(ops)
        c.pages = pages
        assert torch.equal(out[:bad], clean[:bad]) and torch.equal(out[n:], clean[n:])
        assert not torch.isfinite(out[bad:n].float()).any()
        for g in range(nkv):
            assert torch.equal(c.of(scores_out, 0, g), c.of(scores_clean, 0, g)) and torch.equal(c.of(scores_out, 1, g), c.of(scores_clean, 1, g))


def test_no_room_at_all_for_moves(ops):
    from nanohybrid_vlm_b200.kernels.library import KernelError
    p = Pool([64, 10], 1, 16, seed=2)
    p.random(False)
    p.select(ops, [64, 10], [64, 10], 0, 0, room=0)         # nobody is over the budget
    ops.raise_wait_errors()
    p.select(ops, [64, 10], [0, 10], 0, 0, room=0)          # nothing stays: no moves either
    ops.raise_wait_errors()
    births = [torch.arange(n, dtype=torch.int32).view(1, -1) + 5 for n in (64, 10)]
    p.fill([torch.arange(n).float().view(1, -1) for n in (64, 10)], births)     # the best keys stand last
    p.select(ops, [64, 10], [63, 10], 0, 0, room=0)
    with pytest.raises(KernelError, match="key_eviction"):
        ops.raise_wait_errors()
    ops.raise_wait_errors()


# ---------------------------------------------------------------- sizes beyond what the tcgen05 kernels reach
def test_a_pool_of_more_rows_than_a_32_bit_coordinate_reaches(ops):
    """bfloat16 heads of 8: the pool's rows pass 2^31.  A request of many rows beside one of few, scores in place."""
    c = Case([24, 1], [90, 70], 4, 2, 8, 64, torch.bfloat16, seed=21)
    n_pages = 2 ** 31 // (2 * 2 * 64) + 5
    shift = n_pages - c.n_pages
    where = torch.tensor([i if i % 2 else i + shift for i in range(c.n_pages)])
    pages = torch.empty(n_pages, *c.pages.shape[1:], dtype=torch.bfloat16, device="cuda")
    scores, births = torch.empty(n_pages, 2, 64, device="cuda"), torch.empty(n_pages, 2, 64, dtype=torch.int32, device="cuda")
    pages[where], scores[where], births[where] = c.pages.cuda(), c.scores.cuda(), c.births.cuda()
    table = torch.where(c.table >= 0, where[c.table.long().clamp(min=0)].int(), c.table).cuda()
    out = torch.full_like(c.q, math.nan).cuda()
    ops.attention_scored(out, c.q.cuda(), pages, scores, table, c.cu_t, c.lens_t, 2, 1, 24, 90, 4, 2, 8, c.scale, births=births,
                         positions=i32(c.positions))
    ops.raise_wait_errors()
    c.check(out.cpu(), scores[where].cpu(), births[where].cpu())


def test_more_tiles_of_rows_than_a_grid_has_places(ops):
    """53,000 requests of one token with 64 query heads: more tiles of rows than the tcgen05 kernels' grid has."""
    S, nq, d, page, L = 53000, 64, 8, 8, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(S, nq * d, generator=g, device="cuda").bfloat16()
    pages = torch.randn(S, 2, 1, page, d, generator=g, device="cuda").bfloat16()
    scores = torch.rand(S, 1, page, generator=g, device="cuda")
    table = torch.randperm(S, generator=g, device="cuda").int().view(S, 1)
    out, after = torch.empty_like(q), torch.zeros_like(scores)
    ops.attention_scored(out, q, pages, scores, table, torch.arange(S + 1, dtype=torch.int32, device="cuda"),
                         torch.full((S,), L, dtype=torch.int32, device="cuda"), S, 1, 1, L, nq, 1, d, d ** -0.5, scores_out=after)
    ops.raise_wait_errors()
    at = table[:, 0].long()
    k, v = pages[at, 0, 0, :L].double(), pages[at, 1, 0, :L].double()
    p = torch.softmax(q.view(S, nq, d).double() @ k.transpose(1, 2) * d ** -0.5, -1)
    unit = 2 * 2 ** -8 + 2 ** -15                           # the weights and the output, each rounded once; the 32-bit sums
    assert ((out.view(S, nq, d).double() - p @ v).abs() <= p @ v.abs() * unit).all()
    old = scores[at, 0, :L].double()
    old[:, L - 1:] = 0
    assert torch.allclose(after[at, 0, :L].double(), old + p.sum(1), rtol=2 ** -15, atol=0)
    assert (after[:, :, L:] == 0).all()


@pytest.mark.parametrize("new", [1, 40])
def test_queries_that_are_one_row_for_all_tokens(ops, new):
    """q with rows no distance apart: what no copy by tiles can describe is done without it."""
    c = Case([new, 1], [90, 70], 4, 2, 64, 64, torch.bfloat16, seed=23)
    c.q[:] = c.q[:1].clone()
    first, second = c.q[:1].cuda().expand(c.q.shape[0], -1), torch.full_like(c.q, math.nan).cuda()
    scores, births = c.scores.cuda(), c.births.cuda()
    ops.attention_scored(second, first, c.pages.cuda(), scores, c.table.cuda(), c.cu_t, c.lens_t, 2, 1, new, 90, 4, 2, 64, c.scale, births=births,
                         positions=i32(c.positions))
    ops.raise_wait_errors()
    c.check(second.cpu(), scores.cpu(), births.cpu())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page", [(4, 2, 64, 64), (8, 1, 33, 7)])
@pytest.mark.parametrize("news,most", [([1, 4, 0, 1], 2), ([40, 200, 1, 0], 100), ([1, 90, 1, 1], 30)])
def test_requests_that_bring_more_than_was_said_are_left_out(ops, dtype, nq, nkv, d, page, news, most):
    c = Case(news, [300, 250, 70, 20], nq, nkv, d, page, dtype, seed=25)
    want, want_scores, want_births = c.run(ops)
    out, scores, births = torch.full_like(c.q, 9.0).cuda(), c.scores.cuda(), c.births.cuda()
    ops.attention_scored(out, c.q.cuda(), c.pages.cuda(), scores, c.table.cuda(), c.cu_t, c.lens_t, 4, min(news), most, 300, nq, nkv, d, c.scale,
                         births=births, positions=i32(c.positions))
    ops.raise_wait_errors()
    out, scores, births = out.cpu(), scores.cpu(), births.cpu()
    big = slice(news[0], news[0] + news[1])
    assert (out[big] == 9.0).all()
    assert torch.equal(c.of(scores, 1, 0).nan_to_num(-1.0), c.of(c.scores, 1, 0).nan_to_num(-1.0)) and torch.equal(c.of(births, 1, 0), c.of(c.births, 1, 0))
    rest = torch.ones(c.q.shape[0], dtype=torch.bool)
    rest[big] = False
    unit = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -18      # the same sums in other parts: a rounding of the output, or of 32-bit sums
    assert torch.allclose(out[rest].double(), want[rest].double(), rtol=unit, atol=unit)
    for s in (0, 2, 3):
        for g in range(nkv):
            assert torch.allclose(c.of(scores, s, g), c.of(want_scores, s, g), rtol=2.0 ** -15, atol=0) and torch.equal(c.of(births, s, g), c.of(want_births, s, g))


def test_an_output_over_the_queries_is_refused(ops):
    """The second pass reads the queries again: in place the weights would be those of the outputs."""
    from nanohybrid_vlm_b200.kernels.library import KernelError
    c = Case([40, 1], [60, 30], 4, 2, 64, 64, torch.bfloat16, seed=27)
    q, scores = c.q.cuda(), c.scores.cuda()
    with pytest.raises(KernelError, match="memory of its own"):
        ops.attention_scored(q, q, c.pages.cuda(), scores, c.table.cuda(), c.cu_t, c.lens_t, 2, 1, 40, 60, 4, 2, 64, c.scale)
    assert torch.equal(q.cpu(), c.q) and torch.equal(scores.cpu().nan_to_num(-1.0), c.scores.nan_to_num(-1.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page", [(16, 2, 128, 64), (64, 1, 64, 8), (33, 1, 40, 7)])
def test_bounds_above_what_a_step_without_new_tokens_brings(ops, dtype, nq, nkv, d, page):
    c = Case([0, 0, 0], [90, 0, 33], nq, nkv, d, page, dtype, seed=29)
    scores, births = c.scores.cuda(), c.births.cuda()
    q = torch.empty(0, nq * d, dtype=dtype, device="cuda")
    ops.attention_scored(torch.empty_like(q), q, c.pages.cuda(), scores, c.table.cuda(), c.cu_t, c.lens_t, 3, 0, 60, 90, nq, nkv, d, c.scale, births=births,
                         positions=i32([]))
    ops.raise_wait_errors()
    assert torch.equal(scores.cpu().nan_to_num(-1.0), c.scores.nan_to_num(-1.0)) and torch.equal(births.cpu(), c.births)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page,copies", [(4, 2, 128, 64, 1), (3, 1, 40, 24, 1), (20, 4, 96, 16, 1), (2, 2, 64, 64, 100), (8, 1, 256, 32, 60)])
def test_a_query_that_is_no_number_weighs_on_no_key_that_it_does_not_see(ops, dtype, nq, nkv, d, page, copies):
    """Few tokens a request, of few requests (one launch) and of many (two): keys behind the token's own do not notice."""
    n = 4 if nq // nkv < 8 else 1
    c = Case([n, 1] * copies, [40 + n, 30] * copies, nq, nkv, d, page, dtype, seed=31)
    _, clean, _ = c.run(ops)
    q = c.q.clone()
    q[c.cu[0]] = math.nan                                   # the first request's first token
    out, scores, _ = c.run(ops, q=q)
    assert torch.isnan(out[0].float()).all() and not torch.isnan(out[1:].float()).any()
    for g in range(nkv):
        got, want = c.of(scores, 0, g), c.of(clean, 0, g)
        assert torch.isnan(got[:41]).all() and torch.equal(got[41:], want[41:])
        for s in range(1, 2 * copies):
            assert torch.equal(c.of(scores, s, g), c.of(clean, s, g))
