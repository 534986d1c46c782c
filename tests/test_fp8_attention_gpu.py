"""``attention_fp8`` against its definition in 64 bits.

The tolerance of an output element, from arithmetic, with u the output type's unit roundoff
(2^-8 bf16, 2^-11 fp16) and p the weights of its row:

* the output is rounded once: u |o|;
* weights are rounded to fp16 for the second product: 2^-11 sum p |v| (those under the smallest
  normal number are at most 2^-14 / 2^7 of the largest and off by 2^-25 / 2^7 of it at most, and so,
  with n keys, n 2^-32 max |v| in all); exponentials by the hardware's 2^x (2^-22) and sums of n
  terms in fp32 add less than 2^-16 sum p |v|;
* a logit is off by d = scale (2^-17 max |q| sum |k| + D 2^-23 sum |q k|): queries enter as parts of
  8 bits that leave at most 2^-10 of a unit of which their largest element has 224 or more, products are
  summed in fp32; plus 2^-22 |logit| for its scaling. Weights then change by a factor within
  exp(+-2 d) of one another, and the output by (exp(2 d) - 1) sum p |v| at most.
"""

import math

import pytest
import torch

from dropkv_b200 import attention_fp8, tree_mask_from_parents

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Case:
    """A paged cache in 8 bits with drawn contents, NaN in all that no token may see."""

    def __init__(self, Hq, Hkv, D, lens, T, block, dtype, seed=0, spread=1, nhd=False, max_blocks=None, q_scale=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        h = torch.Generator().manual_seed(seed)
        self.B, self.Hq, self.Hkv, self.D, self.T, self.block, self.lens = len(lens), Hq, Hkv, D, T, block, lens
        need = [-(-(n + T) // block) for n in lens]
        self.max_blocks = max_blocks if max_blocks is not None else max(max(need), 1)
        pages = sum(need) + 2
        order = torch.randperm(pages, generator=h).tolist()
        table = torch.full((self.B, self.max_blocks), -1, dtype=torch.int32)
        shape = (pages, block, Hkv, D) if nhd else (pages, Hkv, block, D)
        made = []
        for _ in "KV":
            x = torch.randn(pages, Hkv, block, D, generator=g, device="cuda")
            s = torch.exp2(torch.randint(-spread - 5, spread - 4, (pages, Hkv), generator=g, device="cuda").float())
            x8 = (x / s[..., None, None]).clamp(-448, 448).to(E4M3)
            made.append([x8.view(torch.uint8), s])
        unused = torch.ones(pages, block, dtype=torch.bool)
        for b, n in enumerate(need):
            ids = [order.pop() for _ in range(n)]
            table[b, :min(n, self.max_blocks)] = torch.tensor(ids[:self.max_blocks], dtype=torch.int32)
            for t in range(lens[b] + T):
                unused[ids[t // block], t % block] = False
        for m in made:  # rows past the sequences, and whole pages and scales of none
            m[0].masked_fill_(unused.cuda()[:, None, :, None], 0x7f)
            m[1].masked_fill_(unused.all(1).cuda()[:, None], float("nan"))
        (k, self.ks), (v, self.vs) = made
        self.K, self.V = ((x.transpose(1, 2).contiguous().transpose(1, 2) if nhd else x).view(E4M3) for x in (k, v))
        assert tuple(self.K.shape) == (pages, Hkv, block, D) and shape
        self.table = table.cuda()
        self.cache_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.Q = (q_scale * torch.randn(self.B, T, Hq, D, generator=g, device="cuda")).to(dtype).transpose(1, 2)

    def seen(self, mask, window, sinks, b):
        """[T, keys] what each token sees of the rows that the table holds."""
        n, T = self.lens[b], self.T
        keys = min(n + T, self.max_blocks * self.block)
        j, i = torch.arange(keys), torch.arange(T)
        if mask is None:
            place = n + i
            see = j[None, :] <= place[:, None]
            near = j[None, :] > (place - (window or 0))[:, None]
        else:
            m = (mask if mask.dim() == 2 else mask[b]).cpu()
            place = n + (m.sum(-1) - 1).clamp(min=0)
            see = torch.cat([torch.ones(T, n, dtype=torch.bool), m], 1)[:, :keys]
            near = (j[None, :] > (place - (window or 0))[:, None]) | (j >= n)[None, :]
        if window:
            see = see & (near | (j < sinks)[None, :])
        page = self.table[b].long().cpu()[j // self.block] if keys else j
        return see & ((page >= 0) & (page < self.K.shape[0]))[None, :]

    def check(self, mask=None, window=None, sinks=0, scale=None, out=None, nan_ok=False):
        got = attention_fp8(self.Q, self.K, self.V, self.ks, self.vs, self.cache_lens, self.table, tree_mask=mask,
                            window=window, sinks=sinks, scale=scale) if out is None else out
        assert got.dtype == self.Q.dtype and got.is_contiguous()
        c, u, g = scale or self.D ** -0.5, U[self.Q.dtype], self.Hq // self.Hkv
        for b in range(self.B):
            see = self.seen(mask, window, sinks, b).cuda()
            keys = see.shape[1]
            page = self.table[b].long()[torch.arange(keys, device="cuda") // self.block].clamp(0, self.K.shape[0] - 1)
            row = torch.arange(keys, device="cuda") % self.block
            for h in range(self.Hkv):
                def rows(x, s):
                    y = x.view(torch.uint8)[page, h, row].view(E4M3).double() * s[page, h].double()[:, None]
                    return y.masked_fill(~see.any(0)[:, None], 0.0)
                k, v = rows(self.K, self.ks), rows(self.V, self.vs)
                q = self.Q[b, h * g:(h + 1) * g].double()                       # [g, T, D]
                z = c * q @ k.T
                off = c * (2.0 ** -17 * q.abs().amax(-1, keepdim=True) * k.abs().sum(-1)
                           + self.D * 2.0 ** -23 * q.abs() @ k.abs().T) + 2.0 ** -22 * z.abs()
                off = (off * see).amax(-1, keepdim=True) if keys else torch.zeros(g, self.T, 1).cuda()
                z = z.masked_fill(~see, -math.inf)
                p = torch.softmax(z, -1).masked_fill(~see, 0.0).nan_to_num(0.0)
                want, size = p @ v, p @ v.abs()
                top = v.abs().amax() if keys else 0.0
                tol = u * want.abs() + (2.0 ** -11 + 2.0 ** -16 + torch.expm1(2 * off)) * size + keys * 2.0 ** -32 * top + 2.0 ** -25
                err = (got[b, h * g:(h + 1) * g].double() - want).abs()
                assert bool((err <= tol).all()), (b, h, float((err / tol).nan_to_num(1e9).max()), float(err.max()))
        return got


def tree(T, seed, B=None):
    h = torch.Generator().manual_seed(seed)
    par = torch.tensor([[-1 if i == 0 else int(torch.randint(max(-1, i - 9), i, (1,), generator=h)) for i in range(T)]
                        for _ in range(B or 1)])
    mask = tree_mask_from_parents(par)[0].cuda()
    return mask if B else mask[0]


HEADS = [(32, 8, 128), (28, 4, 128), (14, 2, 64), (8, 8, 128), (16, 1, 64), (5, 1, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("block", [8, 16, 64, 256])
def test_single_tokens(heads, block, dtype):
    Case(*heads, [0, 1, 300, 127, 2000, 129], 1, block, dtype, seed=1).check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,T", [((8, 8, 128), 2), ((8, 8, 64), 8), ((32, 8, 128), 4), ((14, 2, 64), 2), ((8, 8, 128), 16),
                                     ((32, 8, 128), 5), ((28, 4, 128), 33), ((16, 2, 64), 64), ((8, 1, 128), 200),
                                     ((32, 8, 128), 130), ((6, 2, 64), 301)])
def test_chains(heads, T, dtype):
    Case(*heads, [0, 700, 63, 64], T, 32, dtype, seed=2).check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,T,block", [((8, 8, 128), 7, 16), ((8, 8, 64), 16, 8), ((32, 8, 128), 64, 64), ((14, 2, 64), 31, 16),
                                           ((28, 4, 128), 256, 128), ((4, 4, 128), 1, 16)])
def test_trees(heads, T, block, dtype):
    c = Case(*heads, [0, 513, 40], T, block, dtype, seed=3)
    c.check(mask=tree(T, 4, 3))
    c.check(mask=tree(T, 5).transpose(0, 1).contiguous().transpose(0, 1))
    c.check(mask=torch.ones(T, T, dtype=torch.bool, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,T,block", [((8, 8, 128), 1, 16), ((14, 2, 64), 2, 8), ((32, 8, 128), 4, 64), ((28, 4, 128), 50, 32),
                                           ((8, 8, 128), 300, 64), ((32, 8, 64), 129, 256)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (100, 4), (64, 130), (513, 0), (4000, 4), ((1 << 31) - 1, 1 << 31)])
def test_windows_and_sinks(heads, T, block, window, sinks, dtype):
    Case(*heads, [0, 1500, 99, 640], T, block, dtype, seed=6).check(window=window, sinks=sinks)


@pytest.mark.parametrize("heads,T", [((8, 8, 128), 9), ((32, 8, 128), 40)])
@pytest.mark.parametrize("window,sinks", [(40, 0), (100, 4), (700, 1000)])
def test_windows_over_trees(heads, T, window, sinks):
    Case(*heads, [5, 900, 0], T, 16, torch.bfloat16, seed=7).check(mask=tree(T, 8, 3), window=window, sinks=sinks)


@pytest.mark.parametrize("T", [1, 5, 40])
def test_nodes_that_see_nothing_or_little(T):
    c = Case(4, 2, 64, [0, 0, 30], T, 16, torch.bfloat16, seed=9)
    mask = torch.zeros(T, T, dtype=torch.bool, device="cuda")
    got = c.check(mask=mask)
    assert got[:2].abs().max() == 0 and got[2].abs().max() > 0
    mask[T - 1, 0] = True
    c.check(mask=mask)
    c.check(mask=mask, window=T, sinks=0)


@pytest.mark.parametrize("T", [1, 3, 100])
def test_missing_pages_and_short_tables(T):
    c = Case(8, 2, 128, [300, 200, 17], T, 16, torch.float16, seed=10)
    c.table[0, 3:7] = -1
    c.table[0, 12] = c.K.shape[0]
    c.table[0, 13] = (1 << 31) - 1
    c.table[1] = -1
    c.check()
    c.check(window=150, sinks=60)
    assert c.check()[1].abs().max() == 0
    short = Case(8, 2, 128, [300, 40, 64], T, 16, torch.bfloat16, seed=11, max_blocks=4)  # caches past the table's end
    short.check()
    short.check(window=20, sinks=3)  # a window of which nothing is left


@pytest.mark.parametrize("T", [1, 4, 60])
def test_lengths_below_zero_and_past_the_table(T):
    c = Case(8, 2, 64, [0, 64], T, 16, torch.bfloat16, seed=12, max_blocks=4)
    c.cache_lens[0] = -5
    c.check()
    c.cache_lens[1] = (1 << 31) - 1   # more rows than the table holds: what fits is seen
    c.lens[1] = 64
    c.check()
    empty = attention_fp8(c.Q, c.K, c.V, c.ks, c.vs, c.cache_lens, c.table[:, :0])
    assert empty.abs().max() == 0
    none = attention_fp8(c.Q, c.K[:0], c.V[:0], c.ks[:0], c.vs[:0], c.cache_lens, c.table)
    assert none.abs().max() == 0


@pytest.mark.parametrize("T", [1, 2, 8, 50, 300])
def test_values_that_are_no_numbers_reach_only_those_who_see_them(T):
    """NaN in V's rows of late tokens, and of rows out of some tokens' window: NaN in those columns of the
    tokens that see them, and nowhere else. NaN in K: in all columns of those."""
    for what in "VK":
        c = Case(8, 4, 128, [190, 400], T, 16, torch.bfloat16, seed=13)
        clean = c.check(window=100 + T, sinks=2)
        bad = [(0, 190, 5), (0, 190 + T - 1, 127), (1, 400 - 100, 0), (1, 400 - 60, 64), (1, 1, 9), (1, 50, 3)]
        raw = (c.V if what == "V" else c.K).view(torch.uint8)
        want = torch.zeros(c.B, c.Hq, T, c.D, dtype=torch.bool)
        see = [c.seen(None, 100 + T, 2, b) for b in range(2)]
        for b, j, d in bad:
            raw[c.table[b, j // 16].long(), 2, j % 16, d] = 0xff
            want[b, 4:6, :, d if what == "V" else slice(None)] |= see[b][:, j, None] if what == "K" else see[b][:, j]
        got = attention_fp8(c.Q, c.K, c.V, c.ks, c.vs, c.cache_lens, c.table, window=100 + T, sinks=2)
        assert torch.equal(got.isnan().cpu(), want)
        assert torch.equal(got.nan_to_num(0.0)[~want.cuda()], clean[~want.cuda()])


def test_queries_that_are_no_numbers_stay_in_their_rows():
    for T in (1, 3, 70):
        c = Case(8, 2, 64, [100, 3], T, 16, torch.float16, seed=14)
        clean = c.check()
        c.Q[0, 3, T - 1, 7], c.Q[1, 0, 0, 0] = float("nan"), float("inf")
        got = attention_fp8(c.Q, c.K, c.V, c.ks, c.vs, c.cache_lens, c.table)
        want = torch.zeros_like(got, dtype=torch.bool)
        want[0, 3, T - 1] = want[1, 0, 0] = True
        assert torch.equal(got.isnan(), want) and torch.equal(got[~want], clean[~want])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1, 4, 48])
@pytest.mark.parametrize("q_scale,scale,spread", [(1e-3, None, 1), (200.0, 0.01, 1), (12.0, None, 1), (1.0, 3.0, 1), (1.0, None, 6),
                                                  (1.0, 1e-6, 1)])
def test_peaked_and_flat_weights_and_scales_far_apart(T, q_scale, scale, spread, dtype):
    Case(8, 2, 128, [900, 33], T, 16, dtype, seed=15, q_scale=q_scale, spread=spread).check(scale=scale)


@pytest.mark.parametrize("T", [1, 3, 40])
def test_strides_and_alignments_of_queries_and_pages(T):
    c = Case(8, 2, 128, [200, 70], T, 16, torch.bfloat16, seed=16, nhd=True)   # pages by token, then head
    want = c.check()
    q = c.Q
    c.Q = q.contiguous()
    assert torch.equal(c.check(), want)
    wide = torch.zeros(2, 8, T, 131, dtype=q.dtype, device="cuda")
    c.Q = wide[..., 1:129].copy_(q)                                          # rows off 16 bytes
    assert torch.equal(c.check(), want)
    turned = torch.zeros(2, 8, 128, T, dtype=q.dtype, device="cuda").transpose(2, 3)
    c.Q = turned.copy_(q)                                                    # elements apart
    assert torch.equal(c.check(), want)
    c.ks, c.vs = (torch.cat([s, s], 1).t().contiguous().t()[:, :2] for s in (c.ks, c.vs))
    assert torch.equal(c.check(), want)


@pytest.mark.parametrize("T", [1, 2, 20, 200])
def test_many_sequences_and_repeats_are_bitwise_equal(T):
    lens = [(i * 37) % 900 for i in range(70)]
    c = Case(8, 2, 64, lens, T, 16, torch.float16, seed=17)
    first = c.check()
    for _ in range(3):
        again = attention_fp8(c.Q, c.K, c.V, c.ks, c.vs, c.cache_lens, c.table)
        assert torch.equal(first, again)


@pytest.mark.parametrize("T", [1, 6, 64])
def test_one_long_sequence_is_split(T):
    c = Case(32, 8, 128, [30000], T, 64, torch.bfloat16, seed=18)
    c.check()
    c.check(window=9000, sinks=4)


@pytest.mark.parametrize("T", [1, 30])
def test_calls_captured_in_graphs_and_on_streams(T):
    """Two captured calls of one process, replayed on other contents, and calls on two streams at once."""
    cs = [Case(8, 2, 128, [500, 40], T, 16, torch.bfloat16, seed=s) for s in (19, 20)]
    args = lambda c: (c.Q, c.K, c.V, c.ks, c.vs, c.cache_lens, c.table)  # noqa: E731
    graphs, outs = [], []
    for c in cs:
        attention_fp8(*args(c))
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(attention_fp8(*args(c)))
    for c in cs:
        c.Q.mul_(0.5)
        c.cache_lens[0] = 333
        c.lens[0] = 333
    for gr in graphs:
        gr.replay()
    for c, o in zip(cs, outs):
        want = attention_fp8(*args(c))
        assert torch.equal(o, want)
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for c, st in zip(cs, streams):
            with torch.cuda.stream(st):
                got.append(attention_fp8(*args(c)))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, outs[i % 2])
