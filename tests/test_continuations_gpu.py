"""Cache rows, tree attention, beam selection and moves of cached rows against plain evaluations in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HD = 128
F8 = torch.float8_e4m3fn
BOTH = pytest.mark.parametrize("act", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
CACHES = pytest.mark.parametrize("coded", [False, True], ids=["f16", "e4m3"])


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def kernels():
    from blackwell_b200 import kernels
    return kernels


class Store:
    """A cache of M sequences and some layers, filled with random rows (or NaN) and read back in 64 bits."""

    def __init__(self, g, M, layers, nkv, max_seq, coded, fill="random", v_size=1.0):
        shape = (M, layers, nkv, max_seq)
        self.shape, self.coded, self.plane = shape, coded, nkv * max_seq * HD
        x = [torch.empty(shape + (HD,), device="cuda").normal_(generator=g) for _ in range(2)]
        if coded:
            self.k, self.v = [(y * 100).clamp(-448, 448).to(F8) for y in x]
            self.ks = torch.empty(shape, device="cuda").uniform_(0.002, 0.02, generator=g)
            self.vs = torch.empty(shape, device="cuda").uniform_(0.002, 0.02, generator=g) * v_size
        else:
            self.k, self.v = x[0].half(), (x[1] * v_size).half()
            self.ks = self.vs = None
        if fill == "nan":
            for t in (self.k, self.v):
                t.view(torch.uint8).fill_(0x7F if coded else 0x7E)
            if coded:
                self.ks.fill_(math.nan)
                self.vs.fill_(math.nan)

    def args(self, layer=0):
        return kernels().KVCache(self.k, self.v, self.ks, self.vs, self.shape[2], self.shape[3], self.shape[1] * self.plane, layer * self.plane)

    def value(self, layer=0):
        """k, v [M][nkv][max_seq][128] in 64 bits."""
        k, v = self.k[:, layer].double(), self.v[:, layer].double()
        return (k * self.ks[:, layer, ..., None].double(), v * self.vs[:, layer, ..., None].double()) if self.coded else (k, v)

    def bits(self):
        return [t.view(torch.uint8).clone() for t in (self.k, self.v) + ((self.ks, self.vs) if self.coded else ())]


# ------------------------------------------------------------------------------------------------------------------ writing rows
def check_write(M, T, nq, nkv, first, max_seq, coded, act, offset=None, count=None, norms=True, base=1e6, size=1.0, layers=2, layer=1, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    st = Store(g, M, layers, nkv, max_seq, coded)
    qkv = (torch.empty((M, T, nq + 2 * nkv, HD), device="cuda").normal_(generator=g) * size).to(act)
    w = [torch.empty(HD, device="cuda").uniform_(0.5, 1.5, generator=g) for _ in range(2)] if norms else [None, None]
    q = torch.full((M, T, nq, HD), 7.0, dtype=act, device="cuda")
    before, old = st.bits(), st.value(layer)
    kernels().qk_norm_rope_kv_rows(q, st.args(layer), qkv, w[0], w[1], ints(first), None if offset is None else ints(offset),
                                   None if count is None else ints(count), nq, M, T, 1e-6, base)
    x = qkv.double()
    freq = base ** (-torch.arange(0, HD, 2, dtype=torch.float64, device="cuda") / HD)
    after = st.value(layer)
    written = torch.zeros((M, layers, nkv, max_seq), dtype=torch.bool, device="cuda")
    half = torch.finfo(act).eps / 2

    def near(got, want, whole, step):
        # norm (a sum of 128 squares by pairs, rsqrt, two products), angle, sine and cosine to a few units, two products and a sum:
        # under 16 half steps of 32 bits of the row's largest pair, then the rounding of what is stored
        bar = 16 * 2.0 ** -24 * math.sqrt(2) * whole + step
        assert ((got - want).abs() <= bar).all(), ((got - want).abs() / bar).max()

    for m in range(M):
        for i in range(T):
            if first[m] < 0 or (count is not None and i >= count[m]):
                assert (q[m, i] == 7).all()
                continue
            p = first[m] + (offset[m][i] if offset is not None else i)
            c, s = (p * freq).cos(), (p * freq).sin()
            y = x[m, i].clone()
            for lo, hi, wt in ((0, nq, w[0]), (nq, nq + nkv, w[1])):
                if norms:
                    y[lo:hi] = y[lo:hi] / (y[lo:hi].square().mean(-1, keepdim=True) + 1e-6).sqrt() * wt.double()
                a, b = y[lo:hi, 0::2].clone(), y[lo:hi, 1::2].clone()
                y[lo:hi, 0::2], y[lo:hi, 1::2] = a * c - b * s, a * s + b * c
            top = y.abs().amax(-1, keepdim=True)
            near(q[m, i].double(), y[:nq], top[:nq], y[:nq].abs() * half if act == torch.bfloat16 else 0)
            row = first[m] + i
            if row >= max_seq:
                continue
            written[m, layer, :, row] = True
            for got, want, t in ((after[0][m, :, row], y[nq:nq + nkv], top[nq:nq + nkv]), (after[1][m, :, row], y[nq + nkv:], top[nq + nkv:])):
                if coded:   # half a step of three mantissa bits, or of the smallest codes (2^-9 apart), in units of absmax / 448
                    near(got, want, t, torch.maximum(want.abs() * 2.0 ** -4, t / 448 * 2.0 ** -10) * (1 + 2.0 ** -18))
                else:
                    near(got, want, t, torch.maximum(want.abs() * 2.0 ** -11, torch.full_like(want, 2.0 ** -25)))
    now = st.bits()
    for b, a in zip(before, now):   # every other row is as it was
        rows = b.reshape(M, layers, nkv, max_seq, -1), a.reshape(M, layers, nkv, max_seq, -1)
        assert torch.equal(rows[0][~written], rows[1][~written])


@BOTH
@CACHES
@pytest.mark.parametrize("M, T, nq, nkv", [(1, 1, 32, 8), (3, 5, 28, 4), (2, 7, 3, 3), (1, 200, 8, 1), (40, 1, 64, 8)])
def test_write(cuda, M, T, nq, nkv, coded, act):
    check_write(M, T, nq, nkv, [(11 * m) % 40 for m in range(M)], 300, coded, act)


@BOTH
@CACHES
@pytest.mark.parametrize("M, nq, nkv", [(8, 28, 4), (3, 13, 13), (2, 5, 1), (5, 64, 8), (1, 6, 3), (4, 1, 1), (7, 32, 8)])
def test_write_many_rows(cuda, M, nq, nkv, coded, act):
    """Rows enough that a warp takes four heads (more than 32 rows * heads per SM): warps with heads of every kind, blocks of part of a row,
    skipped rows and sequences, nodes, rows behind the cache's end."""
    T = 32 * torch.cuda.get_device_properties(0).multi_processor_count // (M * (nq + 2 * nkv)) + 3
    g = torch.Generator().manual_seed(T)
    first, count = [(37 * m) % 50 for m in range(M)], [T - (m % 3) * (T // 4) for m in range(M)]
    check_write(M, T, nq, nkv, first, 50 + T, coded, act, layers=1, layer=0)
    if M > 2:
        first[1], count[2] = -1, 0
        off = torch.randint(0, T, (M, T), generator=g).tolist()
        check_write(M, T, nq, nkv, first, T, coded, act, offset=off, count=count, layers=1, layer=0, seed=1)
    else:
        check_write(M, T, nq, nkv, first, T // 2, coded, act, norms=False, layers=1, layer=0, seed=1)


@CACHES
def test_write_trees_counts_and_edges(cuda, coded):
    off = [[0, 1, 1, 2, 2], [0, 0, 0, 1, 3], [0, 1, 2, 3, 4], [0, 0, 1, 1, 1], [0] * 5]
    check_write(5, 5, 8, 2, [0, 17, -1, 28, 31], 32, coded, torch.float32, offset=off, count=[5, 3, 5, 9, 0])
    check_write(3, 4, 8, 2, [30, 2 ** 31 - 2, 100], 32, coded, torch.float32)


@CACHES
def test_write_far_positions_and_sizes(cuda, coded):
    check_write(1, 3, 4, 4, [120000], 120003, coded, torch.float32, layers=1, layer=0)
    check_write(2, 3, 4, 2, [5, 9], 16, coded, torch.float32, norms=False, base=10000.0)
    check_write(2, 3, 4, 2, [5, 9], 16, coded, torch.float32, size=1e-4)
    check_write(2, 3, 4, 2, [5, 9], 16, coded, torch.bfloat16, size=50.0)


def test_write_rows_of_zeros_and_tiny_rows(cuda):
    g = torch.Generator("cuda").manual_seed(1)
    st = Store(g, 1, 1, 1, 4, True, fill="nan")
    qkv = torch.zeros((1, 2, 3, HD), device="cuda")
    qkv[0, 1] = 3e-11
    q = torch.empty((1, 2, 1, HD), device="cuda")
    kernels().qk_norm_rope_kv_rows(q, st.args(), qkv, None, None, ints([1]), None, None, 1, 1, 2, 1e-6, 1e4)
    k, v = st.value()
    assert (k[0, 0, 1:3] == 0).all() and (v[0, 0, 1:3] == 0).all() and (st.ks[0, 0, 0, 1:3] == 1).all() and st.ks[0, 0, 0, 3].isnan()


@BOTH
def test_write_codes_and_scales_of_values_of_any_size(cuda, act):
    """Value rows are neither normed nor turned: up to the largest numbers scales are absmax / 448 to two roundings, and codes nearest to x * (448 /
    absmax), the factor off by two steps of 2^-23 and the product by a rounding."""
    g = torch.Generator("cuda").manual_seed(2)
    st = Store(g, 1, 1, 2, 40, True)
    size = torch.logspace(-9, 38, 40, dtype=torch.float64, device="cuda").float()
    qkv = torch.empty((1, 40, 5, HD), device="cuda").uniform_(-1, 1, generator=g)
    qkv[0, :, :3] = 1.0
    qkv = (qkv * size[:, None, None]).to(act)
    assert bool(qkv.isfinite().all()) and float(qkv.abs().max()) > 2.0 ** 126
    kernels().qk_norm_rope_kv_rows(torch.empty((1, 40, 1, HD), dtype=act, device="cuda"), st.args(), qkv, None, None, ints([0]), None, None, 1, 1, 40, 1e-6, 1e4)
    x = qkv[0, :, 3:].float().transpose(0, 1)
    top = x.abs().amax(-1, keepdim=True)
    unit = top[..., 0].double() / 448
    assert ((st.vs[0, 0].double() - unit).abs() <= unit * 2.0 ** -23).all()
    want = x.double() * 448 / top.double()
    assert ((st.v[0, 0].double() - want).abs() <= torch.maximum(want.abs() * 2.0 ** -4, torch.full_like(want, 2.0 ** -10)) + want.abs() * 2.0 ** -21).all()


# ------------------------------------------------------------------------------------------------------------------ attention
def tree_masks(g, M, T):
    """Ancestor masks of random trees, as Python integers [M][T]."""
    out = []
    for _ in range(M):
        u = torch.rand(T, generator=g)
        bits = []
        for i in range(T):
            p = int(u[i] * (i + 1)) - 1
            bits.append((bits[p] if p >= 0 else 0) | 1 << i)
        out.append(bits)
    return out


def words(masks):
    return torch.tensor([[b - (1 << 64) if b >> 63 else b for b in row] for row in masks], dtype=torch.int64, device="cuda")


def check_attention(*a, **kw):
    """By both kernels, then by the one that the sizes choose."""
    k = kernels()
    try:
        for route in (1, 2):
            k.set_tuning(25, route)
            one_attention(*a, **kw)
    finally:
        k.set_tuning(25, 0)
    return one_attention(*a, **kw)


def one_attention(M, T, nq, nkv, first, max_seq, coded, act, masks=None, count=None, hint=0, layers=1, layer=0, q_size=1.5, v_size=1.0, seed=0,
                    store=None, clean=True, stream=None, call=None):
    g = torch.Generator("cuda").manual_seed(seed)
    st = store or Store(g, M, layers, nkv, max_seq, coded, v_size=v_size)
    q = (torch.empty((M, T, nq, HD), device="cuda").normal_(generator=g) * q_size).to(act)
    out = torch.full((M, T, nq, HD), 7.0, dtype=act, device="cuda")
    n = [T if count is None else max(0, min(T, c)) for c in (count or [T] * M)]
    seen = []
    for m in range(M):
        f = min(first[m], max_seq)
        end = min(first[m] + n[m], max_seq)
        see = torch.zeros((T, max_seq), dtype=torch.bool)
        for i in range(n[m] if first[m] >= 0 else 0):
            see[i, :f] = True
            bits = masks[m][i] if masks is not None else (1 << i + 1) - 1
            for j in range(end - f):
                see[i, f + j] = bool(bits >> j & 1)
        seen.append(see.cuda())
    if clean:   # what nobody sees holds NaN
        for m in range(M):
            for t in (st.k, st.v):
                t.view(torch.uint8)[m, layer, :, ~seen[m].any(0)] = 0x7F if coded else 0x7E
            for t in (st.ks, st.vs) if coded else ():
                t[m, layer, :, ~seen[m].any(0)] = math.nan
    k = kernels()
    scratch = torch.full((k.attention_tree_scratch_bytes(M, 64, nq, nkv, max_seq),), 255, dtype=torch.uint8, device="cuda")   # (whatever kernel)
    a = (out, q, st.args(layer), ints(first), None if masks is None else words(masks), None if count is None else ints(count), hint, nq, M, T, scratch)
    (call or k.attention_tree)(*a)
    kk, vv = st.value(layer)
    kk, vv = kk.nan_to_num(0), vv.nan_to_num(0)
    group = nq // nkv
    for m in range(M):
        if first[m] < 0:
            assert (out[m] == 7).all()
            continue
        assert (out[m, n[m]:] == 7).all()
        if n[m] == 0:
            continue
        see = seen[m][:n[m], None, :]
        x = q[m, :n[m]].double().view(n[m], nkv, group, HD)
        score = torch.einsum("ihgd,htd->ihgt", x, kk[m]) / math.sqrt(HD)
        score = score.masked_fill(~see[:, :, None].expand_as(score), -math.inf)
        p = torch.softmax(score, -1).nan_to_num(0)
        want = torch.einsum("ihgt,htd->ihgd", p, vv[m]).reshape(n[m], nq, HD)
        got = out[m, :n[m]].double()
        assert torch.isfinite(got).all()
        # A score is off by 2^-21 (fp32: operands of 22 bits) or 2^-22 (bf16 operands are exact, 32-bit sums) of sum |q k| / sqrt(128) and by
        # some roundings of its own size; a probability by that, by 2^-22 of exp2 and by its own rounding (2^-22 / 2^-12); sums of 16 products at a
        # time, with 2^-23 each; the result is an average of v.
        size = torch.einsum("ihgd,htd->ihgt", x.abs(), kk[m].abs()).div_(math.sqrt(HD)).masked_fill_(~see[:, :, None].expand_as(score), 0)
        ds = 2.0 ** -21 * size.amax(-1) + 2.0 ** -22 * score.abs().masked_fill(score.isinf(), 0).amax(-1)
        fine = 2.0 ** -12 if act == torch.bfloat16 else 2.0 ** -21
        steps = (first[m] + T) / 16 + 64
        bar = (2 * ds + 2 * fine + steps * 2.0 ** -23).reshape(n[m], nq, 1) * torch.einsum("ihgt,htd->ihgd", p, vv[m].abs()).reshape(n[m], nq, HD).amax(-1, keepdim=True)
        if act == torch.bfloat16:
            bar = bar + want.abs() * 2.0 ** -8
        off = float(((got - want).abs() / bar).nan_to_num(0).max())   # (a bar of zero: nothing but zeros)
        assert off <= 1 and (got[(bar == 0).expand_as(got)] == 0).all(), (m, off)
    return out


@BOTH
@CACHES
@pytest.mark.parametrize("M, T, nq, nkv, top", [
    (1, 1, 32, 8, 1), (1, 1, 32, 8, 700), (5, 1, 28, 4, 300), (3, 1, 4, 4, 90), (2, 1, 48, 3, 1500),      # single tokens
    (2, 2, 8, 8, 65), (3, 4, 32, 8, 400), (2, 8, 28, 4, 1000), (1, 17, 5, 1, 33), (2, 33, 8, 2, 257), (2, 64, 16, 4, 500), (1, 64, 64, 8, 2100)])
def test_attention(cuda, M, T, nq, nkv, top, coded, act):
    g = torch.Generator().manual_seed(T)
    first = [max(0, top - 1 - (m * 61) % top) for m in range(M)]
    check_attention(M, T, nq, nkv, first, top + T + 3, coded, act, masks=tree_masks(g, M, T) if T > 1 else None)


@BOTH
@CACHES
def test_attention_chain_counts_and_slots(cuda, coded, act):
    """No masks: a chain.  Counts of every kind, slots without a sequence, sequences that end at the cache's end."""
    check_attention(7, 6, 12, 4, [0, 5, -1, 44, 47, 60, 2 ** 31 - 1], 50, coded, act, count=[6, 0, 6, 4, 6, 100, -3])
    check_attention(4, 6, 12, 4, [600, 0, -5, 3], 606, coded, act, count=[1, 2, 3, 6], hint=40)


@CACHES
def test_attention_rows_that_see_nothing(cuda, coded):
    out = check_attention(2, 5, 8, 2, [0, 0], 40, coded, torch.float32, masks=[[0, 2, 0, 4, 8], [0, 0, 0, 0, 0]])
    assert (out[1] == 0).all() and (out[0, 0] == 0).all() and (out[0, 1] != 0).any()
    # not itself, later nodes, bits of nodes that do not exist
    check_attention(2, 5, 8, 2, [7, 0], 40, coded, torch.float32, masks=[[16, 1, 0, 31, 2 ** 64 - 1], [2 ** 63 | 1, 2, 2, 4, 2]], count=[5, 3])


@CACHES
@pytest.mark.parametrize("hint", [1, 300, 5000])
def test_attention_any_hint(cuda, coded, hint):
    check_attention(2, 3, 16, 4, [4500, 10], 4700, coded, torch.float32, hint=hint, masks=[[1, 3, 5], [1, 2, 7]])


@CACHES
def test_attention_other_layer_and_long_context(cuda, coded):
    check_attention(2, 4, 8, 2, [300, 20], 320, coded, torch.float32, layers=3, layer=2)
    check_attention(1, 3, 4, 1, [40000], 40010, coded, torch.float32, masks=[[1, 3, 5]])


@BOTH
@CACHES
@pytest.mark.parametrize("q_size, v_size", [(1e-6, 1e-3), (6.0, 100.0), (0.0, 1.0)])
def test_attention_sizes(cuda, q_size, v_size, coded, act):
    check_attention(2, 3, 8, 2, [200, 33], 210, coded, act, q_size=q_size, v_size=v_size)


def test_attention_value_scales_of_all_sizes(cuda):
    """Value scales over twenty decades, growing and falling along the context, and rows of scale zero."""
    g = torch.Generator("cuda").manual_seed(3)
    for order in (1, -1):
        st = Store(g, 1, 1, 2, 400, True)
        st.vs *= torch.logspace(-10, 10, 400, device="cuda")[::order] if order == 1 else torch.logspace(-10, 10, 400, device="cuda").flip(0)
        st.vs[0, 0, :, ::7] = 0
        st.ks[0, 0, :, ::5] = 0
        check_attention(1, 2, 4, 2, [390], 400, True, torch.float32, store=st)


@BOTH
@pytest.mark.parametrize("M, T, nq, nkv, top", [(2, 5, 32, 8, 300), (1, 4, 4, 4, 40), (2, 64, 32, 8, 700), (2, 20, 8, 8, 1500), (3, 64, 32, 4, 5000)])
@pytest.mark.parametrize("weighed", [False, True], ids=["hidden", "light"])
def test_attention_value_scales_that_a_row_does_not_weigh(cuda, M, T, nq, nkv, top, act, weighed):
    """Value scales 2^25 times the others', of nodes that other branches do not see, or of positions whose probability is nothing: the rows keep
    their precision, held to the values that they weigh themselves."""
    g = torch.Generator("cuda").manual_seed(T)
    st = Store(g, M, 1, nkv, top + T, True)
    masks = [[1 << i | (1 if i % 3 == 0 else 0) | (2 if i == T - 1 else 0) for i in range(T)] for _ in range(M)]
    first = [top - 3 * m for m in range(M)]
    for m in range(M):
        st.vs[m, :, :, first[m] + 1] *= 2.0 ** 25
        if weighed:
            for at in (0, 9, top // 2, first[m] - 1):   # scores of some 60 either way
                st.ks[m, :, :, at] = 0.4
                st.vs[m, :, :, at] *= 2.0 ** 25
    check_attention(M, T, nq, nkv, first, top + T, True, act, masks=masks, store=st)


@BOTH
def test_attention_value_scales_that_fall_and_end(cuda, act):
    """Value scales that fall by 2^60 along the context, rows of scale -0 and stretches of scale zero at its start, inside and at its end."""
    for T in (3, 64):
        st = Store(torch.Generator("cuda").manual_seed(T), 2, 1, 4, 900, True)
        st.vs *= 2.0 ** torch.linspace(20, -40, 900, device="cuda")
        st.vs[..., :70] = 0
        st.vs[..., 300:450] = -0.0
        st.vs[..., 5::11] = -0.0
        st.vs[0, ..., 760:] = 0
        check_attention(2, T, 16, 4, [800, 830], 900, True, act, store=st)


@BOTH
@pytest.mark.parametrize("M, T, nq, nkv, top", [(10, 1, 28, 4, 7), (5, 14, 48, 3, 2), (6, 7, 48, 3, 39), (2, 40, 20, 1, 700)])
def test_attention_value_scales_of_zero_where_the_scores_are_largest(cuda, M, T, nq, nkv, top, act):
    """Rows whose values are zero take the probability, but no bits of the others' products."""
    g = torch.Generator("cuda").manual_seed(top)
    k, group = kernels(), nq // nkv
    st = Store(g, M, 1, nkv, top + T, True)
    st.vs[..., ::3] = 0
    st.ks[..., ::3] *= 8                               # scores of some 40 either way
    q = (torch.empty((M, T, nq, HD), device="cuda").normal_(generator=g) * 1.5).to(act)
    kk, vv = st.value()
    x = q.double().view(M, T, nkv, group, HD)
    hide = (torch.arange(top + T, device="cuda") > top + torch.arange(T, device="cuda")[:, None])[:, None]
    s = (torch.einsum("mihgd,mhtd->mhigt", x, kk) / math.sqrt(HD)).masked_fill(hide, -math.inf)
    size = (torch.einsum("mihgd,mhtd->mhigt", x.abs(), kk.abs()) / math.sqrt(HD)).masked_fill(hide, 0).amax(-1, keepdim=True)
    p = torch.softmax(s, -1)
    want, weight = [torch.einsum("mhigt,mhtd->mhigd", p, v) for v in (vv, vv.abs())]
    # As in one_attention: a score is off by 2^-21 of sum |q k| / sqrt(128), a probability by that, by its rounding (2^-21 / 2^-12) and, where the references are
    # some 100 apart, by that of their difference (2^-18); sums of 16 products at a time.  A scale of zero counts as 2^-90: f16 steps of 2^-24 are then
    # 2^-114 of the largest probability, over fewer than 2^10 positions 2^-104.
    fine = 2.0 ** -12 if act == torch.bfloat16 else 2.0 ** -21
    bar = (2 * 2.0 ** -21 * size + 2 * fine + 2.0 ** -18 + ((top + T) / 16 + 64) * 2.0 ** -23) * weight.amax(-1, keepdim=True) + 2.0 ** -104 * vv.abs().amax()
    if act == torch.bfloat16:
        bar = bar + want.abs() * 2.0 ** -8
    try:
        for route in (0, 1, 2):
            k.set_tuning(25, route)
            out = torch.zeros_like(q)
            scratch = torch.empty(k.attention_tree_scratch_bytes(M, T, nq, nkv, top + T), dtype=torch.uint8, device="cuda")
            k.attention_tree(out, q, st.args(), ints([top] * M), None, None, 0, nq, M, T, scratch)
            got = out.double().view(M, T, nkv, group, HD).permute(0, 2, 1, 3, 4)
            assert ((got - want).abs() <= bar).all(), (route, float(((got - want).abs() / bar).max()))
    finally:
        k.set_tuning(25, 0)


@BOTH
@CACHES
@pytest.mark.parametrize("M, T, nq, nkv, top", [(40, 9, 32, 8, 1500), (20, 64, 32, 8, 1200), (23, 13, 28, 4, 2050), (80, 3, 24, 8, 700), (460, 2, 20, 1, 300), (90, 40, 32, 8, 130)])
def test_attention_many_tiles_of_a_block(cuda, M, T, nq, nkv, top, coded, act):
    """Blocks that have whole contexts, several of them, many tiles of each, with and without a line of work."""
    g = torch.Generator().manual_seed(M)
    first = torch.randint(top // 2, top, (M,), generator=g).tolist()
    first[M // 2], first[M // 3] = -1, 0
    check_attention(M, T, nq, nkv, first, top + T, coded, act, masks=tree_masks(g, M, T), count=[T - m % 2 * (T // 3) if m % 7 else 0 for m in range(M)])


@BOTH
@CACHES
@pytest.mark.parametrize("T", [5, 64])
def test_attention_scores_and_values_that_grow(cuda, T, coded, act):
    """The maximum and the values' scale move at many places of a long context, up or down."""
    g = torch.Generator("cuda").manual_seed(T)
    M, nq, nkv, top = 22, 32, 8, 1100
    for falling in (False, True):
        st = Store(g, M, 1, nkv, top + T, coded)
        at = torch.linspace(0, 1, top + T, device="cuda")
        at = at.flip(0) if falling else at
        if coded:
            st.ks *= 0.05 + 3 * at
            st.vs *= 2 ** (at * 20 - 10)
        else:
            st.k *= (0.05 + 3 * at)[:, None].half()
            st.v *= 2 ** (at * 10 - 5)[:, None].half()
        check_attention(M, T, nq, nkv, [top - 31 * m for m in range(M)], top + T, coded, act, store=st, clean=False)


@CACHES
def test_attention_shares_of_long_contexts(cuda, coded):
    """More shares than a cluster has blocks where there are heads enough for every SM."""
    check_attention(10, 2, 16, 16, [20000 - 7 * m if m % 3 else 3000 for m in range(10)], 20100, coded, torch.float32)
    if coded:
        check_attention(19, 1, 8, 8, [33000 + m for m in range(19)], 34000, coded, torch.float32)


@BOTH
@pytest.mark.parametrize("M, T, nq, nkv, top", [(1, 1, 32, 8, 1500), (32, 1, 32, 8, 3000), (3, 4, 32, 4, 900), (2, 32, 8, 8, 40000), (2, 33, 8, 8, 700),
                                                (4, 64, 32, 8, 2000), (1, 9, 16, 1, 60000)])
def test_attention_scratch_of_the_size_given(cuda, M, T, nq, nkv, top, act):
    """Scratch of the size that the library gives for the call, whichever kernel takes it."""
    k = kernels()

    def call(out, q, cache, first, mask, count, hint, nq, M, T, _):
        n = k.attention_tree_scratch_bytes(M, T, nq, nkv, top + T)
        k.attention_tree(out, q, cache, first, mask, count, hint, nq, M, T, torch.full((n,), 255, dtype=torch.uint8, device="cuda"))

    check_attention(M, T, nq, nkv, [top - 17 * m for m in range(M)], top + T, True, act, call=call)


@CACHES
@pytest.mark.parametrize("M, T, nq, nkv, top", [(2, 1, 8, 2, 40000), (1, 3, 28, 4, 33000), (1, 40, 8, 2, 40000), (1, 64, 16, 2, 20000)])
def test_attention_root_mean_square_of_long_contexts(cuda, M, T, nq, nkv, top, coded):
    """The largest error may grow with the number of sums; the root mean square hardly does, and shows a probability of fewer bits."""
    g = torch.Generator("cuda").manual_seed(T)
    k, group = kernels(), nq // nkv
    st = Store(g, M, 1, nkv, top + T, coded)
    q = torch.empty((M, T, nq, HD), device="cuda").normal_(generator=g)
    kk, vv = st.value()
    s = torch.einsum("mihgd,mhtd->mhigt", q.double().view(M, T, nkv, group, HD), kk) / math.sqrt(HD)
    size = float(torch.einsum("mihgd,mhtd->mhigt", q.abs().view(M, T, nkv, group, HD), kk.abs().float()).amax()) / math.sqrt(HD)
    s.masked_fill_((torch.arange(top + T, device="cuda") > top + torch.arange(T, device="cuda")[:, None])[:, None], -math.inf)
    want = torch.einsum("mhigt,mhtd->mihgd", torch.softmax(s, -1), vv).reshape(M, T, nq, HD)
    del s
    try:
        for route in (0, 1, 2):
            k.set_tuning(25, route)
            out = torch.zeros_like(q)
            scratch = torch.empty(k.attention_tree_scratch_bytes(M, T, nq, nkv, top + T), dtype=torch.uint8, device="cuda")
            k.attention_tree(out, q, st.args(), ints([top] * M), None, None, 0, nq, M, T, scratch)
            # A probability is off by 2^-20 and, twice, by what its score is (2^-21 of sum |q k| / sqrt(128)); rounded sums of 16 positions walk: sqrt(n / 16)
            # steps of 2^-23.  P in 11 bits alone would be 2^-12 / sqrt(3) = 1.4e-4.
            bar = 2.0 ** -20 * (1 + size) + math.sqrt(top / 16) * 2.0 ** -23
            off = float((out.double() - want).square().mean().sqrt() / want.square().mean().sqrt())
            assert off <= bar and bar < 5e-5, (route, off, bar)
    finally:
        k.set_tuning(25, 0)


def test_attention_far_offsets(cuda):
    """Sequences whose rows lie beyond 2^32 bytes and elements."""
    g = torch.Generator("cuda").manual_seed(4)
    k = kernels()
    small = Store(g, 2, 1, 2, 300, True)
    stride = (1 << 32) + 128 * 7
    rows = stride // 128 + 2 * 300
    kv = [torch.empty((rows, HD), dtype=F8, device="cuda") for _ in range(2)]
    sc = [torch.empty(rows, device="cuda") for _ in range(2)]
    for big, s in zip(kv + sc, (small.k, small.v, small.ks, small.vs)):
        s = s.view(torch.uint8) if s.dtype == F8 else s
        big = big.view(torch.uint8) if big.dtype == F8 else big
        big[:600] = s[0].reshape((600,) + big.shape[1:])
        big[stride // 128:] = s[1].reshape((600,) + big.shape[1:])
    c = k.KVCache(kv[0], kv[1], sc[0], sc[1], 2, 300, stride)
    q = torch.randn((2, 3, 4, HD), generator=g, device="cuda")
    outs = []
    for cache in (small.args(), c):
        out = torch.zeros_like(q)
        k.attention_tree(out, q, cache, ints([290, 250]), None, None, 0, 4, 2, 3, None)
        outs.append(out)
    assert torch.equal(*outs)
    qkv = torch.randn((2, 1, 8, HD), generator=g, device="cuda")
    for cache in (small.args(), c):
        k.qk_norm_rope_kv_rows(torch.empty((2, 1, 4, HD), device="cuda"), cache, qkv, None, None, ints([5, 295]), None, None, 4, 2, 1, 0.0, 1e4)
    assert torch.equal(kv[0].view(torch.uint8)[stride // 128:], small.k[1].view(torch.uint8).reshape(600, HD))
    assert torch.equal(sc[1][stride // 128:], small.vs[1].reshape(600))


@CACHES
@pytest.mark.parametrize("T, nq", [(4, 16), (60, 32)])
def test_attention_same_bits_again_and_in_graphs(cuda, coded, T, nq):
    """Repeated calls, a captured one that is replayed with other positions, and calls on two streams at once."""
    g = torch.Generator("cuda").manual_seed(5)
    k = kernels()
    M, nkv = 2, 4
    st = Store(g, M, 1, nkv, 2100, coded)
    q = torch.randn((M, T, nq, HD), generator=g, device="cuda")
    first, out = ints([2000, 700]), torch.zeros((M, T, nq, HD), device="cuda")
    new = lambda: torch.empty(k.attention_tree_scratch_bytes(M, T, nq, nkv, 2100), dtype=torch.uint8, device="cuda")  # noqa: E731
    scratch, cache = new(), st.args()
    k.attention_tree(out, q, cache, first, None, None, 0, nq, M, T, scratch)
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k.attention_tree(out, q, cache, first, None, None, 0, nq, M, T, scratch)
    for pos in ([2000, 700], [64, 1999], [2000, 700]):
        first.copy_(ints(pos))
        graph.replay()
        eager = torch.zeros_like(out)
        k.attention_tree(eager, q, cache, first, None, None, 0, nq, M, T, new())
        assert torch.equal(eager, out)
    assert torch.equal(out, want)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [torch.zeros_like(out) for _ in range(2)]
    work = [new(), new()]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, o, w in zip(streams, outs, work):
            k.attention_tree(o, q, cache, first, None, None, 0, nq, M, T, w, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ------------------------------------------------------------------------------------------------------------------ beam selection
def check_select(logits, score, ended, eos, keep, M, B, stride=None, inplace=False):
    V = logits.shape[1]
    k = kernels()
    parent, token = torch.full((M, keep), 99, dtype=torch.int32, device="cuda"), torch.full((M, keep), 99, dtype=torch.int32, device="cuda")
    s_in, e_in = score.clone(), None if ended is None else ended.clone()
    s_out = s_in if inplace else torch.full((M, keep), 99.0, device="cuda")
    e_out = e_in if inplace else torch.full((M, keep), 99, dtype=torch.uint8, device="cuda")
    scratch = torch.full((k.beam_select_scratch_bytes(V, B, keep, M),), 255, dtype=torch.uint8, device="cuda")
    full = logits
    if stride:
        full = torch.full((M * B, stride), math.nan, device="cuda")
        full[:, :V] = logits
    k.beam_select(parent, token, s_out, e_out, full, stride or V, V, s_in, e_in, eos, B, keep, M, scratch)
    x = torch.where(logits.isnan(), -math.inf, logits).double().view(M, B, V)
    x = (score.double()[..., None] + torch.log_softmax(x, -1)).nan_to_num(-math.inf, math.inf, -math.inf)
    if ended is not None:
        own = torch.full((V,), -math.inf, dtype=torch.float64, device="cuda")
        for m, b in ended.bool().nonzero().tolist():
            x[m, b] = own
            x[m, b, eos] = score[m, b].double()
    val, at = x.view(M, -1).sort(dim=1, descending=True, stable=True)
    if val.shape[1] < keep:
        pad = keep - val.shape[1]
        val, at = torch.nn.functional.pad(val, (0, pad), value=-math.inf), torch.nn.functional.pad(at, (0, pad))
    val, at = val[:, :keep], at[:, :keep]
    none = val == -math.inf
    wp, wt = torch.where(none, -1, at // V), torch.where(none, -1, at % V)
    assert torch.equal(parent.long(), wp) and torch.equal(token.long(), wt)
    # exp2 of 32 bits in the log-sums (2^-21 of an argument under 2^5), then the rounding to 32 bits
    assert torch.equal(s_out.isinf(), none)
    fine = ~none
    assert ((s_out.double() - val)[fine].abs() <= val[fine].abs() * 2.0 ** -24 + 2.0 ** -20).all()
    gone = (wt == eos) & fine
    if ended is not None:
        gone |= fine & ended.bool().gather(1, wp.clamp(min=0))
    assert torch.equal(e_out.bool(), gone)


@pytest.mark.parametrize("M, B, V, keep", [(1, 1, 1, 1), (1, 1, 7, 10), (2, 4, 1000, 4), (1, 4, 32768, 8), (3, 7, 2049, 14), (2, 8, 151643, 8), (1, 64, 5000, 64), (9, 16, 4099, 16), (1, 16, 11000, 32), (4, 2, 90001, 3),
                                           (20, 16, 8193, 32), (1, 2, 300000, 1)])
def test_select(cuda, M, B, V, keep):
    g = torch.Generator("cuda").manual_seed(V + keep)
    logits = torch.empty((M * B, V), device="cuda").normal_(generator=g) * 2
    score = -torch.rand((M, B), generator=g, device="cuda") * 3
    check_select(logits, score, None, -1, keep, M, B)
    ended = (torch.rand((M, B), generator=g, device="cuda") < 0.4).to(torch.uint8)
    check_select(logits, score, ended, min(2, V - 1), keep, M, B, stride=V + 5)
    if keep == B:
        check_select(logits, score, ended, min(2, V - 1), keep, M, B, inplace=True)


@pytest.mark.parametrize("keep", [1, 5, 64])
def test_select_equal_and_few_values(cuda, keep):
    """Many equal logits (more than are ranked at once), rows of few values, nothing left."""
    g = torch.Generator("cuda").manual_seed(keep)
    B, V = 3, 20000
    score = torch.tensor([[-1.0, -1.0, -1.0]], device="cuda")
    check_select(torch.zeros((B, V), device="cuda"), score, None, -1, keep, 1, B)
    steps = torch.randint(0, 3, (B, V), generator=g, device="cuda").float()
    check_select(steps.repeat(2, 1), score.repeat(2, 1), None, 5, keep, 2, B)
    some = torch.full((B, V), -math.inf, device="cuda")
    some[0, 17], some[2, 17], some[2, 19999] = 1.0, 3.0, 3.0
    check_select(some, score, None, 17, keep, 1, B)
    many = torch.where(torch.rand((B, V), generator=g, device="cuda") < 0.2, steps, -math.inf)
    many[1] = -math.inf
    check_select(many, score, None, -1, keep, 1, B)
    check_select(torch.arange(V, device="cuda").float().div(V / 8).repeat(B, 1), score, None, -1, keep, 1, B)
    check_select(torch.arange(V, 0, -1, device="cuda").float().div(V / 8).repeat(B, 1), score, None, -1, keep, 1, B)


def test_select_dead_beams_and_odd_values(cuda):
    g = torch.Generator("cuda").manual_seed(9)
    B, V = 4, 3000
    logits = torch.empty((2 * B, V), device="cuda").normal_(generator=g)
    score = torch.tensor([[0.0, -math.inf, -math.inf, -math.inf], [-2.0, -math.inf, -0.5, -1.0]], device="cuda")   # the first step of a search
    check_select(logits, score, None, 7, 4, 2, B)
    check_select(logits, score, torch.tensor([[1, 1, 0, 0], [0, 1, 1, 1]], dtype=torch.uint8, device="cuda"), 7, 8, 2, B)
    logits[0, ::3] = math.nan
    logits[5] = -math.inf
    logits[6, 1] = -3e38
    logits[7, 5] = 1e30
    check_select(logits, score, None, 7, 4, 2, B)
    logits[4, 9] = math.inf
    check_select(logits, score, None, 7, 4, 2, B)


@pytest.mark.parametrize("keep", [1, 4, 20])
@pytest.mark.parametrize("V", [50, 9001])
def test_select_zeros_of_both_signs(cuda, V, keep):
    """-0 and +0 are equal: the lower token first, inside a stretch of a row and across them."""
    g = torch.Generator("cuda").manual_seed(V)
    B = 2
    logits = -torch.empty((2 * B, V), device="cuda").normal_(generator=g).abs().round()
    logits = torch.where((logits == 0) & (torch.rand((2 * B, V), generator=g, device="cuda") < 0.5), 0.0, logits)
    logits[:, 0], logits[:, 1] = -1.0, -0.0
    assert bool((logits.view(torch.int32) == -2 ** 31).any()) and bool((logits.view(torch.int32) == 0).any())
    check_select(logits, torch.tensor([[-1.0, -1.5], [-3.0, -0.25]], device="cuda"), None, -1, keep, 2, B)


def test_select_scores_of_both_zeros(cuda):
    """Beams that have ended with -0 and +0: the lower beam first."""
    logits, score = torch.zeros((3, 40), device="cuda"), torch.tensor([[-0.0, 0.0, -0.0]], device="cuda")
    check_select(logits, score, torch.ones((1, 3), dtype=torch.uint8, device="cuda"), 7, 3, 1, 3)
    check_select(logits, score, torch.ones((1, 3), dtype=torch.uint8, device="cuda"), 7, 1, 1, 3)


@pytest.mark.parametrize("V", [60, 20000])
def test_select_equal_scores_of_ended_beams_whose_logits_are_nothing(cuda, V):
    """Beams that have ended with the same score: their logits are not looked at, whatever their bits."""
    logits = torch.empty((4, V), device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(V))
    logits[1:3].view(torch.int32).fill_(-1)             # NaN with every bit set
    score = torch.tensor([[-40.0, -1.5, -1.5, -60.0]], device="cuda")
    for keep in (1, 2, 4, 9):
        check_select(logits, score, torch.tensor([[0, 1, 1, 0]], dtype=torch.uint8, device="cuda"), 7, keep, 1, 4)


@pytest.mark.parametrize("B, V, keep", [(1, 300, 5), (2, 30000, 6), (1, 200000, 40), (8, 151643, 8), (16, 40000, 20)])
def test_select_logits_closer_than_their_scores(cuda, B, V, keep):
    """Scores that fall together in 64 bits: within a beam the larger logit first, wherever in the row; equal logits by token."""
    g = torch.Generator("cuda").manual_seed(V)
    k = kernels()
    logits = torch.empty((B, V), device="cuda").normal_(generator=g) * 1e-20
    logits[:, V // 3], logits[:, V - 2], logits[:, 5] = 9e-20, 9e-20, 8e-20
    score = -torch.arange(B, device="cuda").float()[None]
    assert len(set((score[0, :1].double() + (logits[0].double() - math.log(V))).tolist())) == 1
    parent, token = torch.zeros((1, keep), dtype=torch.int32, device="cuda"), torch.zeros((1, keep), dtype=torch.int32, device="cuda")
    out = torch.zeros((1, keep), device="cuda")
    scratch = torch.empty(k.beam_select_scratch_bytes(V, B, keep, 1), dtype=torch.uint8, device="cuda")
    k.beam_select(parent, token, out, None, logits, V, V, score, None, -1, B, keep, 1, scratch)
    assert (parent == 0).all() and torch.equal(token[0].long(), logits[0].sort(descending=True, stable=True).indices[:keep])


def test_select_in_a_graph(cuda):
    g = torch.Generator("cuda").manual_seed(10)
    k, B, V = kernels(), 4, 9000
    logits, score = torch.randn((B, V), generator=g, device="cuda"), torch.zeros((1, B), device="cuda")
    out = [torch.zeros((1, B), dtype=torch.int32, device="cuda") for _ in range(2)] + [torch.zeros((1, B), device="cuda")]
    scratch = torch.empty(k.beam_select_scratch_bytes(V, B, B, 1), dtype=torch.uint8, device="cuda")
    call = lambda o: k.beam_select(o[0], o[1], o[2], None, logits, V, V, score, None, 0, B, B, 1, scratch)  # noqa: E731
    call(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for _ in range(3):
        logits.normal_(generator=g)
        graph.replay()
        got = [o.clone() for o in out]
        call(out)
        assert all(torch.equal(a, b) for a, b in zip(got, out))


# ------------------------------------------------------------------------------------------------------------------ moving rows
@CACHES
@pytest.mark.parametrize("M, B, layers, nkv, max_seq", [(1, 1, 1, 1, 5), (2, 4, 2, 3, 50), (1, 9, 3, 2, 130), (3, 32, 1, 1, 20), (2, 5, 2, 8, 700)])
def test_reorder(cuda, M, B, layers, nkv, max_seq, coded):
    g = torch.Generator("cuda").manual_seed(B)
    st = Store(g, M * B, layers + 1, nkv, max_seq, coded)
    for turn in range(3):
        parent = torch.randint(-1, B + 1, (M, B), generator=g, device="cuda", dtype=torch.int32) if turn else torch.arange(B - 1, -1, -1, device="cuda", dtype=torch.int32).repeat(M, 1)
        lo = ints([m % 3 for m in range(M)]) if turn else None
        hi = ints([max_seq + 9 if m % 2 else max_seq - 2 - m for m in range(M)])
        want = st.bits()
        for w in want:
            rows = w.view(M, B, layers + 1, nkv, max_seq, -1)
            old = rows.clone()
            for m in range(M):
                for b in range(B):
                    p = int(parent[m, b])
                    a, z = (int(lo[m]) if lo is not None else 0), min(int(hi[m]), max_seq)
                    if 0 <= p < B:
                        rows[m, b, 1:, :, a:z] = old[m, p, 1:, :, a:z]
        kernels().kv_reorder(st.args(1), parent, lo, hi, B, M, layers, st.plane)
        assert all(torch.equal(a, b) for a, b in zip(want, st.bits()))


@CACHES
def test_reorder_of_nothing(cuda, coded):
    st = Store(torch.Generator("cuda").manual_seed(1), 4, 1, 2, 30, coded)
    before = st.bits()
    kernels().kv_reorder(st.args(), ints([[1, 0], [1, 0]]), ints([9, -4]), ints([9, -1]), 2, 2, 1, st.plane)
    kernels().kv_reorder(st.args(), ints([[1, 0], [1, 0]]), ints([2 ** 31 - 1, 1]), ints([-2 ** 31, 1 - 2 ** 31]), 2, 2, 1, st.plane)
    kernels().kv_reorder(st.args(), ints([[0, 1], [0, 1]]), None, ints([30, 30]), 2, 2, 1, st.plane)
    assert all(torch.equal(a, b) for a, b in zip(before, st.bits()))


@CACHES
def test_layers_around_sequences(cuda, coded):
    """A cache [layer][sequence]: rows moved between beams and along paths, and one layer's attention."""
    g = torch.Generator("cuda").manual_seed(12)
    k, L, M, B, nkv, top = kernels(), 3, 2, 3, 2, 40
    st = Store(g, L, M * B, nkv, top, coded)
    sides = [t.view(torch.uint8) for t in (st.k, st.v) + ((st.ks, st.vs) if coded else ())]
    rows = lambda t: t.view(L, M, B, nkv, top, -1)  # noqa: E731
    before = [rows(t).clone() for t in sides]
    cache = lambda layer: k.KVCache(st.k, st.v, st.ks, st.vs, nkv, top, st.plane, layer * M * B * st.plane)  # noqa: E731
    k.kv_reorder(cache(0), ints([[1, 2, 0], [2, 1, 2]]), ints([4, 0]), ints([17, 33]), B, M, L, M * B * st.plane)
    for m, (parents, lo, hi) in enumerate((((1, 2, 0), 4, 17), ((2, 1, 2), 0, 33))):
        for t, old in zip(sides, before):
            want = old[:, m].clone()
            want[:, :, :, lo:hi] = old[:, m][:, list(parents), :, lo:hi]
            assert torch.equal(rows(t)[:, m], want)
    now = [rows(t).clone() for t in sides]
    k.kv_keep_rows(cache(1), ints([5] * 6), ints([[0, 2, 3]] * 6), ints([3] * 6), M * B, 3, L - 1, M * B * st.plane)
    for t, old in zip(sides, now):
        want = old.clone()
        want[1:, :, :, :, 5:8] = old[1:, :, :, :, [5, 7, 7]]   # (path 3 is not inside 0 .. T - 1)
        assert torch.equal(rows(t), want)
    q = torch.randn((M * B, 2, 4, HD), generator=g, device="cuda")
    outs = [torch.zeros_like(q) for _ in range(2)]
    k.attention_tree(outs[0], q, cache(2), ints([30] * 6), None, None, 0, 4, M * B, 2, None)
    k.attention_tree(outs[1], q, k.KVCache(st.k[2], st.v[2], st.ks[2] if coded else None, st.vs[2] if coded else None, nkv, top, st.plane), ints([30] * 6),
                     None, None, 0, 4, M * B, 2, None)
    assert torch.equal(*outs) and bool(outs[0].any())


@CACHES
def test_sequences_that_share_a_cache(cuda, coded):
    """batch_elems 0: every sequence reads the same rows."""
    g = torch.Generator("cuda").manual_seed(13)
    k, M, nkv, top = kernels(), 5, 2, 300
    st = Store(g, 1, 1, nkv, top, coded)
    q = torch.randn((M, 3, 4, HD), generator=g, device="cuda")
    out, one = torch.zeros_like(q), torch.zeros_like(q)
    for n, o in ((M, out), (1, one)):
        for m in range(0, M, n):
            k.attention_tree(o[m:m + n], q[m:m + n], k.KVCache(st.k, st.v, st.ks, st.vs, nkv, top, 0), ints([290] * n), None, None, 0, 4, n, 3, None)
    assert torch.equal(out, one) and bool(out.any())


@CACHES
@pytest.mark.parametrize("M, T, layers, nkv", [(1, 1, 1, 1), (1, 8, 5, 8), (3, 7, 2, 3), (5, 64, 2, 2), (2, 33, 3, 1)])
def test_keep_rows(cuda, M, T, layers, nkv, coded):
    g = torch.Generator("cuda").manual_seed(T)
    max_seq = 2 * T + 6
    st = Store(g, M, layers + 1, nkv, max_seq, coded)
    for turn in range(4):
        path = torch.randint(-1 if turn else 0, T + (1 if turn else 0), (M, T), generator=g, device="cuda", dtype=torch.int32)
        if turn == 0:
            path = path.sort(1).values.int()
        first = [(3, -1, T + 4, 0, 2 ** 31 - 1)[(m + turn) % 5] for m in range(M)]
        count = [(T, T // 2, T + 5, -1, 1)[(m + turn) % 5] for m in range(M)]
        want = st.bits()
        for w in want:
            rows = w.view(M, layers + 1, nkv, max_seq, -1)
            old = rows.clone()
            for m in range(M):
                for i in range(min(T, count[m])):
                    p = int(path[m, i])
                    if first[m] >= 0 and 0 <= p < T and first[m] + max(p, i) < max_seq:
                        rows[m, 1:, :, first[m] + i] = old[m, 1:, :, first[m] + p]
        kernels().kv_keep_rows(st.args(1), ints(first), path, ints(count), M, T, layers, st.plane)
        assert all(torch.equal(a, b) for a, b in zip(want, st.bits()))


# ------------------------------------------------------------------------------------------------------------------ together
@CACHES
def test_a_drafted_tree_is_verified_and_kept(cuda, coded):
    """A prompt is written, a tree of six nodes drafted, attended and one path accepted; the next token's attention over what is kept has
    the bits of one over a cache into which the path's tokens were written one after the other."""
    g = torch.Generator("cuda").manual_seed(6)
    k = kernels()
    M, nq, nkv, max_seq, T, n = 2, 8, 2, 60, 6, [31, 17]
    a, b = Store(g, M, 1, nkv, max_seq, coded), Store(g, M, 1, nkv, max_seq, coded, fill="nan")
    b.k.copy_(a.k), b.v.copy_(a.v)
    if coded:
        b.ks.copy_(a.ks), b.vs.copy_(a.vs)
    w = [torch.empty(HD, device="cuda").uniform_(0.5, 1.5, generator=g) for _ in range(2)]
    prompt = torch.randn((M, 31, nq + 2 * nkv, HD), generator=g, device="cuda")
    q = torch.empty((M, 31, nq, HD), device="cuda")
    for st in (a, b):
        k.qk_norm_rope_kv_rows(q, st.args(), prompt, w[0], w[1], ints([0, 0]), None, ints(n), nq, M, 31, 1e-6, 1e6)
    depth = [[0, 1, 1, 2, 2, 3], [0, 0, 1, 1, 2, 3]]
    masks = [[1, 3, 5, 11, 21, 43], [1, 2, 5, 10, 21, 53]]
    path, count = [[0, 2, 4, 0, 0, 0], [0, 2, 4, 5, 0, 0]], [3, 4]
    nodes = torch.randn((M, T, nq + 2 * nkv, HD), generator=g, device="cuda")
    qt = torch.empty((M, T, nq, HD), device="cuda")
    k.qk_norm_rope_kv_rows(qt, a.args(), nodes, w[0], w[1], ints(n), ints(depth), None, nq, M, T, 1e-6, 1e6)
    check = torch.zeros((M, T, nq, HD), device="cuda")
    k.attention_tree(check, qt, a.args(), ints(n), words(masks), None, 0, nq, M, T, None)
    k.kv_keep_rows(a.args(), ints(n), ints(path), ints(count), M, T, 1, a.plane)
    for i in range(4):   # the same tokens one by one; the first sequence has three
        now = [n[0] + i if i < 3 else -1, n[1] + i]
        one = torch.stack([nodes[0, path[0][min(i, 2)]], nodes[1, path[1][i]]])
        q1, out = torch.zeros((M, nq, HD), device="cuda"), torch.zeros((M, nq, HD), device="cuda")
        k.qk_norm_rope_kv_rows(q1, b.args(), one, w[0], w[1], ints(now), None, None, nq, M, 1, 1e-6, 1e6)
        k.attention_tree(out, q1, b.args(), ints(now), None, None, 0, nq, M, 1, None)
        for m in range(M):
            if now[m] >= 0:   # (another order of the sums: 32-bit roundings)
                assert torch.equal(q1[m], qt[m, path[m][i]])
                assert torch.allclose(out[m], check[m, path[m][i]], rtol=0, atol=2.0 ** -17 * float(check.abs().max()))
    for m in range(M):
        end = n[m] + count[m]
        assert torch.equal(a.k.view(torch.uint8)[m, 0, :, :end], b.k.view(torch.uint8)[m, 0, :, :end])
    ends = [n[m] + count[m] for m in range(M)]
    last = torch.randn((M, 1, nq + 2 * nkv, HD), generator=g, device="cuda")
    outs = []
    for st in (a, b):
        q1, out = torch.empty((M, nq, HD), device="cuda"), torch.empty((M, nq, HD), device="cuda")
        k.qk_norm_rope_kv_rows(q1, st.args(), last, w[0], w[1], ints(ends), None, None, nq, M, 1, 1e-6, 1e6)
        k.attention_tree(out, q1, st.args(), ints(ends), None, None, 0, nq, M, 1, None)
        outs.append(out)
    assert torch.equal(*outs)


def test_beams_share_a_prompt_and_part(cuda):
    """Beams over one cache each: selection, reordering, the next row; every beam's cache is its parent's plus its own token."""
    g = torch.Generator("cuda").manual_seed(7)
    k = kernels()
    B, nq, nkv, max_seq, V, L = 4, 4, 2, 40, 500, 2
    st = Store(g, B, L, nkv, max_seq, True)
    table = torch.randn((V, nq + 2 * nkv, HD), generator=g, device="cuda")
    score = torch.tensor([[0.0, -math.inf, -math.inf, -math.inf]], device="cuda")
    ended = torch.zeros((1, B), dtype=torch.uint8, device="cuda")
    parent, token = torch.zeros((1, B), dtype=torch.int32, device="cuda"), torch.zeros((1, B), dtype=torch.int32, device="cuda")
    scratch = torch.empty(k.beam_select_scratch_bytes(V, B, B, 1), dtype=torch.uint8, device="cuda")
    tokens = [[] for _ in range(B)]
    for step in range(6):
        logits = torch.randn((B, V), generator=g, device="cuda")
        k.beam_select(parent, token, score, ended, logits, V, V, score, ended, 3, B, B, 1, scratch)
        k.kv_reorder(st.args(), parent, ints([10]), ints([10 + step]), B, 1, L, st.plane)
        tokens = [tokens[int(parent[0, b])] + [int(token[0, b])] for b in range(B)]
        for layer in range(L):
            q = torch.empty((B, 1, nq, HD), device="cuda")
            k.qk_norm_rope_kv_rows(q, st.args(layer), table[token[0].long()], None, None, ints([10 + step] * B), None, None, nq, B, 1, 1e-6, 1e4)
    again = Store(g, B, L, nkv, max_seq, True)
    for b in range(B):
        rows = table[torch.tensor(tokens[b], device="cuda")]
        q = torch.empty((1, 6, nq, HD), device="cuda")
        one = Store(g, 1, 1, nkv, max_seq, True)
        k.qk_norm_rope_kv_rows(q, one.args(), rows, None, None, ints([10]), None, None, nq, 1, 6, 1e-6, 1e4)
        for layer in range(L):
            assert torch.equal(one.k.view(torch.uint8)[0, 0, :, 10:16], st.k.view(torch.uint8)[b, layer, :, 10:16])
            assert torch.equal(one.vs[0, 0, :, 10:16], st.vs[b, layer, :, 10:16])
    del again


@CACHES
@pytest.mark.parametrize("T, nq", [(3, 8), (40, 32)])
def test_whole_steps_captured_and_replayed(cuda, T, nq, coded):
    """A tree's step (rows, attention, accepted path) and a beam's (selection, reordering, rows, attention) in one graph, replayed with other positions,
    masks, paths and logits: the bits of the same calls one after the other."""
    g = torch.Generator("cuda").manual_seed(T)
    k, M, B, L, nkv, top, V = kernels(), 2, 3, 2, 4, 500, 3000
    a, b = Store(g, M * B, L, nkv, top, coded), Store(g, M * B, L, nkv, top, coded)
    for x, y in zip((a.k, a.v) + ((a.ks, a.vs) if coded else ()), (b.k, b.v) + ((b.ks, b.vs) if coded else ())):
        y.copy_(x)
    N = M * B
    tree, token = torch.empty((N, T, nq + 2 * nkv, HD), device="cuda"), torch.empty((N, 1, nq + 2 * nkv, HD), device="cuda")
    logits, first, offset = torch.empty((N, V), device="cuda"), ints([0] * N), torch.zeros((N, T), dtype=torch.int32, device="cuda")
    mask, path, count, lo = torch.zeros((N, T), dtype=torch.int64, device="cuda"), torch.zeros((N, T), dtype=torch.int32, device="cuda"), ints([0] * N), ints([0] * M)
    hi, score0 = ints([0] * M), torch.zeros((M, B), device="cuda")

    def buffers():
        one = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
        return dict(q=one(N, T, nq, HD), o=one(N, T, nq, HD), q1=one(N, 1, nq, HD), o1=one(N, 1, nq, HD), parent=one(M, B, dtype=torch.int32), token=one(M, B, dtype=torch.int32),
                    score=one(M, B), w=one(k.attention_tree_scratch_bytes(N, T, nq, nkv, top), dtype=torch.uint8), w2=one(k.beam_select_scratch_bytes(V, B, B, M), dtype=torch.uint8))

    def step(st, z):
        for layer in range(L):
            k.qk_norm_rope_kv_rows(z["q"], st.args(layer), tree, None, None, first, offset, None, nq, N, T, 1e-6, 1e4)
            k.attention_tree(z["o"], z["q"], st.args(layer), first, mask, None, 0, nq, N, T, z["w"])
        k.kv_keep_rows(st.args(), first, path, count, N, T, L, st.plane)
        k.beam_select(z["parent"], z["token"], z["score"], None, logits, V, V, score0, None, -1, B, B, M, z["w2"])
        k.kv_reorder(st.args(), z["parent"], lo, hi, B, M, L, st.plane)
        for layer in range(L):
            k.qk_norm_rope_kv_rows(z["q1"], st.args(layer), token, None, None, first, None, None, nq, N, 1, 1e-6, 1e4)
            k.attention_tree(z["o1"], z["q1"], st.args(layer), first, None, None, 0, nq, N, 1, z["w"])

    def inputs(seed):
        h = torch.Generator().manual_seed(seed)
        for x in (tree, token, logits):
            x.normal_(generator=g)
        first.copy_(torch.randint(0, top - T, (N,), generator=h))
        offset.copy_(torch.randint(0, T, (N, T), generator=h))
        mask.copy_(words(tree_masks(h, N, T)))
        path.copy_(torch.randint(0, T, (N, T), generator=h).sort(1).values)
        count.copy_(torch.randint(0, T + 1, (N,), generator=h))
        lo.copy_(torch.randint(0, 100, (M,), generator=h))
        hi.copy_(torch.randint(0, top + 1, (M,), generator=h))
        score0.copy_(-torch.rand((M, B), generator=h))

    za, zb = buffers(), buffers()
    inputs(0)
    step(a, za)
    step(b, zb)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a, za)
    for seed in range(1, 5):
        inputs(seed)
        graph.replay()
        graph.replay()
        for _ in range(2):
            step(b, zb)
        assert all(torch.equal(za[n], zb[n]) for n in ("q", "o", "q1", "o1", "parent", "token", "score"))
        assert all(torch.equal(x, y) for x, y in zip(a.bits(), b.bits()))


# ------------------------------------------------------------------------------------------------------------------ refusals of the tensors
def test_refused_tensors(cuda):
    k = kernels()
    st = Store(torch.Generator("cuda").manual_seed(8), 2, 1, 2, 16, True)
    q = torch.zeros((2, 1, 4, HD), device="cuda")
    with pytest.raises(ValueError):
        k.KVCache(st.k, st.v, None, None, 2, 16, st.plane)
    with pytest.raises(ValueError):
        k.KVCache(st.k, st.v, st.ks[:1], st.vs, 2, 16, st.plane)
    for bad in ((2, 16, -HD), (2, 16, st.plane, -HD), (0, 16, st.plane), (2, 0, st.plane)):
        with pytest.raises(ValueError):
            k.KVCache(st.k, st.v, st.ks, st.vs, *bad)
    with pytest.raises(ValueError):
        k.kv_reorder(st.args(), ints([0, 0]), None, ints([4]), 2, 1, 1, -HD)
    ok = (q, q, st.args(), ints([0, 0]), None, None, 0, 4, 2, 1, None)
    k.attention_tree(*ok)
    for i, bad in ((0, q[:1]), (0, q.half()), (1, q.transpose(0, 2)), (3, torch.zeros(2, device="cuda")), (3, torch.zeros(2, dtype=torch.int32)), (4, ints([0, 0])),
                   (8, 3)):
        with pytest.raises(ValueError):
            k.attention_tree(*ok[:i], bad, *ok[i + 1:])
    with pytest.raises(k.KernelError):
        k.attention_tree(q, q, st.args(), ints([0, 0]), None, None, 0, 3, 2, 1, None)
    with pytest.raises(ValueError):
        k.kv_reorder(st.args(), ints([0, 0, 0]), None, ints([4]), 3, 1, 1, st.plane)
