"""GPU tests of the serving operators against plain implementations in 64 bits.

Tolerances (u = eps/2 is the largest relative rounding error of the 16-bit type, A = the softmax-weighted mean of |v|):
* attention: every probability is rounded once to 16 bits for the second product (u A), the result once (u |o|).  A score is
  a sum of D exact products in 32 bits and is scaled and exponentiated in 32 bits, so it is off by at most
  S = (D + 8) 2^-24 max(sum_d |q_d k_d| scale, 1), which moves numerator and denominator by that factor each (2 S A).  The
  second product is accumulated 16 keys at a time in 32 bits, at worst truncating (N/16 2^-23 A); the smallest fp16
  probabilities fall below the type's normal range: off by 2^-25 where the largest is at least 2^7 (N 2^-32 max|v|).
  Errors of second order: 2 % on top.
* lse: S for the largest score, N 2^-24 for a serial sum, and a few roundings of a number of its size.
* rotary: the angle's reduced form has a relative error of 2^-24, sine and cosine (2 units in the last place), their scaling,
  two products and a sum (3 more roundings): below 16 2^-24 (|a| + |b|) m in all; then one rounding, u |result|."""
import math
import os
import subprocess

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def ftg():
    import ft_gemm_b200
    ft_gemm_b200.load()
    assert torch.cuda.is_available()
    return ft_gemm_b200


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _offsets(lengths):
    return torch.tensor([0] + list(np.cumsum(lengths)), dtype=torch.int32, device="cuda")


def _half_eps(dtype):
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------- attention against 64 bits
def _check_rows(out, lse, q, k, v, visible, scale):
    """One sequence: q, out [n, H, D], k, v [m, Hkv, D], visible [n, m], lse [n, H]."""
    n, heads, dim = q.shape
    m, kv_heads, _ = k.shape
    group = heads // kv_heads
    for h in range(heads if n else 0):
        if m:
            kd, vd = k[:, h // group].double(), v[:, h // group].double()
            qd = q[:, h].double()
            vd = torch.where(visible.any(0)[:, None], vd, 0.0)  # what nobody sees does not count
            kd = torch.where(visible.any(0)[:, None], kd, 0.0)
            x = (qd @ kd.T) * scale
            size = ((qd.abs() @ kd.abs().T) * scale).max().item()
            x = x.masked_fill(~visible, -math.inf)
            top = x.amax(-1, keepdim=True)
            e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
            total = e.sum(-1, keepdim=True)
            p = e / torch.where(total == 0, 1.0, total)
            want, weight, biggest = p @ vd, p @ vd.abs(), vd.abs().max().item()
            want_lse = (torch.where(top == -math.inf, -math.inf, top) + torch.log(total))[:, 0]
        else:
            want, weight, biggest, size = torch.zeros(n, dim, dtype=torch.float64, device=q.device), 0.0, 0.0, 0.0
            want_lse = torch.full((n,), -math.inf, dtype=torch.float64, device=q.device)
        u, s = _half_eps(q.dtype), (dim + 8) * 2.0 ** -24 * max(size, 1.0)
        bound = 1.02 * (u * (want.abs() + weight) + 2 * s * weight + (m / 16) * 2.0 ** -23 * weight + m * 2.0 ** -32 * biggest) + 1e-30
        bound = bound + torch.finfo(q.dtype).smallest_normal * u * 2  # results below the type's normal range
        off = (out[:, h].double() - want).abs()
        assert bool((off <= bound).all()), f"head {h}: off by {off.max().item()} at {off.argmax().item()}, {(off / bound).max().item()} of the bound"
        if lse is not None:
            empty = want_lse == -math.inf
            assert bool((lse[:, h][empty] == -math.inf).all())
            away = (lse[:, h].double() - want_lse)[~empty].abs()
            assert bool((away <= s + m * 2.0 ** -24 + 2.0 ** -21 * (1 + want_lse[~empty].abs())).all())


def _prompt_case(ftg, lengths, heads, kv_heads, dim, dtype, causal=True, key_lengths=None, seed=0, scale=0.0, spare=3, layout="plain", poison=True):
    gen = _gen(seed)
    key_lengths = lengths if key_lengths is None else key_lengths
    t, tk = sum(lengths) + spare, sum(key_lengths) + spare
    if layout == "fused":  # slices of a fused projection
        assert t == tk
        qkv = _randn(gen, (t, heads + 2 * kv_heads, dim), dtype)
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        out = torch.full((heads, t, dim), 7.0, dtype=dtype, device="cuda").transpose(0, 1)
    else:
        q, k, v = _randn(gen, (t, heads, dim), dtype), _randn(gen, (tk, kv_heads, dim), dtype), _randn(gen, (tk, kv_heads, dim), dtype)
        out = torch.full((t, heads, dim), 7.0, dtype=dtype, device="cuda")
    if poison:  # rows behind the last sequence hold anything
        q[sum(lengths):], k[sum(key_lengths):], v[sum(key_lengths):] = math.nan, math.inf, math.nan
    lse = torch.full((t, heads), 7.0, device="cuda")
    op = ftg.PromptAttention(heads, kv_heads, dim, dtype=dtype, causal=causal, scale=scale)
    op.run(q, k, v, out, _offsets(lengths), key_offsets=None if key_lengths is lengths else _offsets(key_lengths), lse=lse)
    op.report()
    a = b = 0
    for n, m in zip(lengths, key_lengths):
        visible = torch.ones(n, m, dtype=torch.bool, device="cuda")
        if causal:
            visible = torch.arange(m, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] + (m - n)
        _check_rows(out[a:a + n], lse[a:a + n], q[a:a + n], k[b:b + m], v[b:b + m], visible, scale or dim ** -0.5)
        a, b = a + n, b + m
    assert bool((out[a:] == 7.0).all()) and bool((lse[a:] == 7.0).all()), "rows behind the last sequence were written"
    return q, k, v, out


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_lengths(ftg, dtype, dim, causal):
    _prompt_case(ftg, [1, 0, 7, 127, 128, 129, 0, 255, 256, 257, 2, 500], 4, 2, dim, DTYPES[dtype], causal)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (5, 1), (7, 1), (12, 2), (16, 1), (20, 4), (33, 1), (64, 1), (100, 1), (128, 1), (24, 8)])
def test_prompt_head_groups(ftg, heads, kv_heads):
    _prompt_case(ftg, [70, 3, 131], heads, kv_heads, 64 if heads % 2 else 128, torch.bfloat16, seed=heads)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_more_or_fewer_keys_than_queries(ftg, dim, causal):
    """Keys in front of the queries; fewer keys than queries leaves rows empty; no keys at all."""
    _prompt_case(ftg, [5, 100, 40, 9, 0, 130, 1], 6, 2, dim, torch.float16, causal, key_lengths=[300, 40, 0, 9, 17, 129, 1000])


def test_prompt_no_keys_at_all(ftg):
    _prompt_case(ftg, [3, 2], 2, 1, 64, torch.bfloat16, True, key_lengths=[0, 0], spare=0)


@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_strided_views(ftg, dim):
    _prompt_case(ftg, [33, 260, 1], 8, 2, dim, torch.bfloat16, layout="fused")


def test_prompt_scale_and_long(ftg):
    _prompt_case(ftg, [2500], 2, 1, 128, torch.bfloat16, scale=0.5)
    _prompt_case(ftg, [1, 5000, 3], 4, 2, 64, torch.float16)


def test_prompt_peaked_scores(ftg):
    """Scores of some hundreds whose maximum keeps moving: the running maximum has to follow."""
    gen = _gen(5)
    n, dtype = 700, torch.bfloat16
    q = _randn(gen, (n, 2, 128), dtype, 4.0)
    ramp = torch.linspace(0.1, 8.0, n, device="cuda")[:, None, None]
    k = (torch.randn((n, 2, 128), generator=gen, device="cuda") * ramp).to(dtype)
    v = _randn(gen, (n, 2, 128), dtype)
    out = torch.empty_like(q)
    op = ftg.PromptAttention(2, 2, 128, dtype=dtype)
    op.run(q, k, v, out, _offsets([n]))
    op.report()
    _check_rows(out, None, q, k, v, torch.ones(n, n, dtype=torch.bool, device="cuda").tril(), 128 ** -0.5)


def test_prompt_neighbours_do_not_leak(ftg):
    """A sequence of NaN and infinities between two others."""
    gen = _gen(6)
    lengths, dtype = [45, 50, 77], torch.float16
    q, k, v = (_randn(gen, (sum(lengths), 2, 64), dtype) for _ in range(3))
    for x, bad in ((q, math.nan), (k, math.inf), (v, math.nan)):
        x[45:95] = bad
    out = torch.empty_like(q)
    for causal in (True, False):
        op = ftg.PromptAttention(2, 2, 64, dtype=dtype, causal=causal)
        op.run(q, k, v, out, _offsets(lengths))
        op.report()
        for a, b in ((0, 45), (95, 172)):
            visible = torch.ones(b - a, b - a, dtype=torch.bool, device="cuda")
            _check_rows(out[a:b], None, q[a:b], k[a:b], v[a:b], visible.tril() if causal else visible, 0.125)
        assert bool(out[45:95].isnan().all())


def test_prompt_offsets_past_32_bits(ftg):
    """Key rows so far apart that element offsets pass 2^32."""
    n, dtype = 90, torch.bfloat16
    gen = _gen(7)
    far = torch.empty((n, 50_000_000), dtype=dtype, device="cuda")
    k, v = far[:, :128].view(n, 2, 64), far[:, 49_000_000:49_000_128].view(n, 2, 64)
    k.copy_(_randn(gen, (n, 2, 64), dtype))
    v.copy_(_randn(gen, (n, 2, 64), dtype))
    q = _randn(gen, (n, 4, 64), dtype)
    out = torch.empty_like(q)
    op = ftg.PromptAttention(4, 2, 64, dtype=dtype)
    op.run(q, k, v, out, _offsets([n]))
    op.report()
    _check_rows(out, None, q, k, v, torch.ones(n, n, dtype=torch.bool, device="cuda").tril(), 0.125)


# ---------------------------------------------------------------- over the cache
def _paged(rng, lengths, page, spare=2):
    need = [-(-n // page) for n in lengths]
    order = rng.permutation(sum(need) + spare)
    table = np.full((len(lengths), max(need + [1]) + 1), -1, dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return sum(need) + spare, table


def _random_mask(rng, drafted, words):
    rows = rng.randint(0, 2 ** 32, (sum(drafted), words), dtype=np.uint64).astype(np.uint32)
    rows[rng.rand(sum(drafted)) < 0.2] = 0  # nothing of the drafted tokens
    return rows


def _tree_case(ftg, contexts, drafted, heads, kv_heads, dim, page, dtype, mask="random", seed=0, by_head=False, layers=2, scale=0.0):
    rng, gen = np.random.RandomState(seed), _gen(seed)
    lengths = [c + n for c, n in zip(contexts, drafted)]
    pages, table = _paged(rng, lengths, page)
    shape = (layers, pages, kv_heads, page, dim) if by_head else (layers, pages, page, kv_heads, dim)
    k, v = torch.full(shape, math.nan, dtype=dtype, device="cuda"), torch.full(shape, math.nan, dtype=dtype, device="cuda")
    if by_head:
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    cache = ftg.PagedCache(k, v)
    layer, plain = layers - 1, []
    for b, m in enumerate(lengths):  # places behind a sequence's end stay NaN
        plain.append((_randn(gen, (m, kv_heads, dim), dtype), _randn(gen, (m, kv_heads, dim), dtype)))
        slots = torch.tensor([int(table[b, i // page]) * page + i % page for i in range(m)], dtype=torch.int64, device="cuda")
        cache.append(layer, *plain[-1], slots)
    t = sum(drafted)
    q = _randn(gen, (t + 2, heads, dim), dtype)
    q[t:] = math.nan
    out, lse = torch.full_like(q, 7.0), torch.full((t + 2, heads), 7.0, device="cuda")
    words = max(1, -(-max(drafted + [1]) // 32)) + seed % 2
    rows = _random_mask(rng, drafted, words)
    packed = torch.zeros((t + 2, words), dtype=torch.int32, device="cuda")
    packed[:t] = torch.from_numpy(rows.view(np.int32)).cuda()
    op = ftg.TreeAttention(heads, cache, scale=scale)
    args = (q, layer, _offsets(drafted), torch.from_numpy(table).cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), out)
    op.run(*args, mask=packed if mask == "random" else None, lse=lse)
    op.report()
    at = 0
    for b, (c, n) in enumerate(zip(contexts, drafted)):
        own = torch.ones(n, n, dtype=torch.bool).tril()
        if mask == "random":
            bits = np.unpackbits(rows[at:at + n].view(np.uint8), axis=1, bitorder="little")[:, :n]
            own = torch.from_numpy(bits.astype(bool)).reshape(n, n)
        visible = torch.cat([torch.ones(n, c, dtype=torch.bool), own], 1).cuda()
        _check_rows(out[at:at + n], lse[at:at + n], q[at:at + n], *plain[b], visible, scale or dim ** -0.5)
        at += n
    assert bool((out[t:] == 7.0).all()) and bool((lse[t:] == 7.0).all()), "rows behind the last sequence were written"


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
def test_tree_pages(ftg, page, dtype):
    """Contexts that end inside a page and a tile, empty ones, empty mask rows, sequences without queries."""
    _tree_case(ftg, [0, 1, 15, 127, 128, 129, 1000, 300, 0], [3, 1, 9, 33, 2, 64, 70, 0, 1], 8, 2, 128 if page != 32 else 64, page, DTYPES[dtype], seed=page)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 1), (15, 3), (32, 8), (7, 1), (128, 1)])
def test_single_tokens(ftg, heads, kv_heads, dim):
    _tree_case(ftg, [0, 5, 126, 127, 128, 700, 2047, 64], [1] * 8, heads, kv_heads, dim, 16, torch.bfloat16, mask=None, seed=heads)


@pytest.mark.parametrize("group", [1, 3, 6, 8])
@pytest.mark.parametrize("mask", ["random", None])
def test_trees_and_chains(ftg, group, mask):
    """Row tiles of one, two and several times 128 rows, chains (pieces of prompts) among them."""
    _tree_case(ftg, [50, 4000, 0, 131], [200, 17, 300, 96], 2 * group, 2, 128, 64, torch.float16, mask=mask, seed=group)


def test_tree_by_head_pages(ftg):
    _tree_case(ftg, [77, 1], [20, 5], 8, 4, 64, 32, torch.bfloat16, by_head=True)


def test_tree_many_sequences(ftg):
    rng = np.random.RandomState(1)
    _tree_case(ftg, [int(x) for x in rng.randint(0, 300, 700)], [int(x) for x in rng.randint(0, 3, 700)], 2, 1, 64, 16, torch.bfloat16)


def test_tree_long_context(ftg):
    _tree_case(ftg, [70000, 10], [6, 2], 4, 1, 128, 64, torch.bfloat16, seed=2)
    _tree_case(ftg, [40000], [40], 16, 2, 64, 128, torch.float16, seed=3)


def test_tree_far_pages(ftg):
    """Pages so far into the cache that element offsets pass 2^32."""
    dtype, page, gen = torch.bfloat16, 16, _gen(9)
    pages = 2_200_000  # of 16 x 1 x 128 elements: 4.5e9
    k, v = (torch.empty((1, pages, page, 1, 128), dtype=dtype, device="cuda") for _ in range(2))
    cache = ftg.PagedCache(k, v)
    ids, m = [pages - 1, 3, pages - 7, 2_100_001], 60
    kk, vv = _randn(gen, (m, 1, 128), dtype), _randn(gen, (m, 1, 128), dtype)
    cache.append(0, kk, vv, torch.tensor([ids[i // page] * page + i % page for i in range(m)], device="cuda"))
    q = _randn(gen, (4, 2, 128), dtype)
    out = torch.empty_like(q)
    op = ftg.TreeAttention(2, cache)
    op.run(q, 0, _offsets([4]), torch.tensor([ids], dtype=torch.int32, device="cuda"), torch.tensor([m], dtype=torch.int32, device="cuda"), out)
    op.report()
    visible = torch.arange(m, device="cuda")[None] <= torch.arange(4, device="cuda")[:, None] + m - 4
    _check_rows(out, None, q, kk, vv, visible, 128 ** -0.5)


def test_tree_bad_pages_read_as_zeros(ftg):
    dtype, gen = torch.bfloat16, _gen(10)
    k, v = (_randn(gen, (1, 4, 16, 2, 64), dtype) for _ in range(2))
    cache = ftg.PagedCache(k, v)
    q = _randn(gen, (1, 4, 64), dtype)
    out = torch.empty_like(q)
    table = torch.tensor([[2, -5, 4, 2 ** 31 - 1, 1]], dtype=torch.int32, device="cuda")
    op = ftg.TreeAttention(4, cache)
    op.run(q, 0, _offsets([1]), table, torch.tensor([75], dtype=torch.int32, device="cuda"), out)
    op.report()
    zeros = torch.zeros((48, 2, 64), dtype=dtype, device="cuda")
    kk, vv = (torch.cat([x[0, 2], zeros, x[0, 1, :11]]) for x in (k, v))
    _check_rows(out, None, q, kk, vv, torch.ones(1, 75, dtype=torch.bool, device="cuda"), 0.125)


def test_lengths_past_the_table_are_cut(ftg):
    """A length that the page table cannot hold reads what the table names and nothing else."""
    dtype, gen = torch.float16, _gen(11)
    k, v = (_randn(gen, (1, 3, 16, 1, 64), dtype) for _ in range(2))
    op = ftg.TreeAttention(2, ftg.PagedCache(k, v))
    q = _randn(gen, (1, 2, 64), dtype)
    out = torch.empty_like(q)
    op.run(q, 0, _offsets([1]), torch.tensor([[2, 0]], dtype=torch.int32, device="cuda"), torch.tensor([40], dtype=torch.int32, device="cuda"), out)
    op.report()
    _check_rows(out, None, q, torch.cat([k[0, 2], k[0, 0]]), torch.cat([v[0, 2], v[0, 0]]), torch.ones(1, 32, dtype=torch.bool, device="cuda"), 0.125)


# ---------------------------------------------------------------- rotary positions and appending
def _rotated(x, positions, frequencies, rotary, interleaved, magnitude, inverse):
    theta = positions.double()[:, None] * torch.tensor(frequencies, dtype=torch.float64, device="cuda")
    c, s = torch.cos(theta)[:, None] * magnitude, torch.sin(theta)[:, None] * magnitude * (-1 if inverse else 1)
    x = x.double()
    y, size = x.clone(), torch.zeros_like(x)
    first = slice(0, rotary, 2) if interleaved else slice(0, rotary // 2)
    second = slice(1, rotary, 2) if interleaved else slice(rotary // 2, rotary)
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(magnitude)
    return y, size


def _check_rotated(got, want, size):
    u = _half_eps(got.dtype)
    bound = u * 1.01 * want.abs() + 16 * 2.0 ** -24 * size + torch.finfo(got.dtype).smallest_normal * u
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by {off.max().item()}, {(off / bound).max().item()} of the bound"


ROTARY = [dict(head_dim=128), dict(head_dim=64, interleaved=True), dict(head_dim=128, rotary_dim=32, scaling="linear", factor=4.0),
          dict(head_dim=64, rotary_dim=48, interleaved=True, scaling="base", factor=8.0), dict(head_dim=96, rotary_dim=96),
          dict(head_dim=128, scaling="by_parts", factor=8.0, original_length=8192, base=500000.0, magnitude=1.25), dict(head_dim=256, rotary_dim=16)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", range(len(ROTARY)))
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary(ftg, case, dtype, inverse):
    o, gen, dtype = ROTARY[case], _gen(case), DTYPES[dtype]
    rotary = ftg.Rotary(**o)
    d, r = o["head_dim"], o.get("rotary_dim", o["head_dim"])
    for tokens, heads, kv_heads in ((1, 1, 1), (65, 6, 2), (500, 40, 0), (37, 3, 1)):
        fused = _randn(gen, (tokens + 1, heads + 2 * kv_heads, d), dtype)
        q, k = fused[:tokens, :heads], fused[:tokens, heads:heads + kv_heads] if kv_heads else None
        positions = torch.randint(0, 3_000_000, (tokens,), generator=gen, device="cuda")
        positions[0] = 0
        q_out = torch.full((tokens, heads, d), 7.0, dtype=dtype, device="cuda")
        k_out = torch.full((kv_heads, tokens, d), 7.0, dtype=dtype, device="cuda").transpose(0, 1) if kv_heads else None
        rotary.run(q, k, positions, q_out, k_out, inverse=inverse)
        for x, y in ((q, q_out), (k, k_out)):
            if x is not None:
                want, size = _rotated(x, positions, rotary.frequencies(), r, o.get("interleaved", False), o.get("magnitude", 1.0), inverse)
                _check_rotated(y, want, size)
                assert torch.equal(y[..., r:], x[..., r:])
        before = fused.clone()
        rotary.run(q, k, positions, q, k, inverse=inverse)  # in place, in a fused projection
        assert torch.equal(q, q_out) and (k is None or torch.equal(k, k_out))
        assert torch.equal(fused[:, heads + kv_heads:], before[:, heads + kv_heads:]) and torch.equal(fused[tokens], before[tokens])


@pytest.mark.parametrize("tokens,heads,kv_heads,d", [(513, 5, 2, 128), (2049, 12, 4, 64), (4096, 32, 8, 128), (4099, 16, 4, 128), (5000, 3, 1, 256),
                                                      (4097, 24, 8, 64), (6001, 1, 1, 16)])
def test_rotary_many_tokens(ftg, tokens, heads, kv_heads, d):
    """Blocks of one, two and three tokens, the last one not full; with the append, q in place, rows of padding among them."""
    gen, dtype = _gen(tokens), torch.bfloat16
    rotary = ftg.Rotary(d)
    q, k, v = (_randn(gen, (tokens, h, d), dtype) for h in (heads, kv_heads, kv_heads))
    positions = torch.randint(0, 200_000, (tokens,), generator=gen, device="cuda")
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    rotary.run(q, k, positions, q_out, k_out)
    for x, y in ((q, q_out), (k, k_out)):
        _check_rotated(y, *_rotated(x, positions, rotary.frequencies(), d, False, 1.0, False))
    if d not in (64, 128):
        return
    pages = -(-tokens // 64) + 1
    cache = ftg.PagedCache.empty(1, pages, 64, kv_heads, d, dtype)
    cache.k.fill_(7.0), cache.v.fill_(7.0)
    slots = torch.randperm(pages * 64, generator=gen, device="cuda")[:tokens]
    slots[::10] = -1
    cache.append(0, k, v, slots, rotary=rotary, positions=positions, q=q, q_out=q)
    assert torch.equal(q, q_out)
    for held, rows in ((cache.k, k_out), (cache.v, v)):
        want = torch.full((pages * 64, kv_heads, d), 7.0, dtype=dtype, device="cuda")
        want[slots[slots >= 0]] = rows[slots >= 0]
        assert torch.equal(held.view(pages * 64, kv_heads, d), want)


def test_rotary_inverse_is_the_gradient(ftg):
    """Against differences: a linear map's derivative along x is the map of x, so <g, R x> = <R^T g, x>, and R^T is `inverse`."""
    gen, n = _gen(3), 50
    for o in (dict(head_dim=64, magnitude=0.5), dict(head_dim=128, rotary_dim=64, interleaved=True)):
        rotary, d = ftg.Rotary(**o), o["head_dim"]
        x, g = _randn(gen, (n, 4, d), torch.float16), _randn(gen, (n, 4, d), torch.float16)
        positions = torch.randint(0, 9999, (n,), generator=gen, device="cuda")
        y, back = torch.empty_like(x), torch.empty_like(x)
        rotary.run(x, None, positions, y)
        rotary.run(g, None, positions, back, inverse=True)
        left, right = (g.double() * y.double()).sum((1, 2)), (back.double() * x.double()).sum((1, 2))
        # each product carries one rounding of y or of back
        bound = 2 ** -11 * 1.05 * ((g.double() * y.double()).abs().sum((1, 2)) + (back.double() * x.double()).abs().sum((1, 2))) + 1e-3
        assert bool(((left - right).abs() <= bound).all())
        # differences: R(x + t e) - R(x) = t R e, element for element, up to the rounding of both sides
        e = torch.zeros_like(x)
        e[:, 1, 3] = 1.0
        up, column = torch.empty_like(x), torch.empty_like(x)
        rotary.run((x + e).to(x.dtype), None, positions, up)
        rotary.run(e, None, positions, column)
        step = ((x + e).to(x.dtype).double() - x.double())[:, 1, 3]
        want = column.double() * step[:, None, None]
        assert bool(((up.double() - y.double() - want).abs() <= 2 ** -11 * 1.05 * (up.double().abs() + y.double().abs() + want.abs()) + 1e-6).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("by_head", [False, True])
def test_append(ftg, dtype, by_head):
    gen, dtype, page, heads, kv_heads, d = _gen(4), DTYPES[dtype], 16, 6, 2, 64
    shape = (3, 9, kv_heads, page, d) if by_head else (3, 9, page, kv_heads, d)
    k_cache, v_cache = _randn(gen, shape, dtype), _randn(gen, shape, dtype)
    if by_head:
        k_cache, v_cache = k_cache.transpose(2, 3), v_cache.transpose(2, 3)
    k_before, v_before = k_cache.clone(), v_cache.clone()
    cache, rotary = ftg.PagedCache(k_cache, v_cache), ftg.Rotary(d, rotary_dim=32)
    tokens = 70
    q, k, v = _randn(gen, (tokens, heads, d), dtype), _randn(gen, (tokens, kv_heads, d), dtype), _randn(gen, (tokens, kv_heads, d), dtype)
    positions = torch.randint(0, 5000, (tokens,), generator=gen, device="cuda")
    slots = torch.randperm(9 * page, generator=gen, device="cuda")[:tokens]
    slots[5], slots[6], slots[7] = -1, 9 * page, -(2 ** 62)  # padding: not written
    q_out = torch.empty_like(q)
    cache.append(1, k, v, slots, rotary=rotary, positions=positions, q=q, q_out=q_out)
    want, size = _rotated(q, positions, rotary.frequencies(), 32, False, 1.0, False)
    _check_rotated(q_out, want, size)
    k_out, unused = torch.empty_like(k), torch.empty_like(q)
    rotary.run(q, k, positions, unused, k_out)
    written = [i for i in range(tokens) if i not in (5, 6, 7)]
    for i in written:
        page_i, place = divmod(int(slots[i]), page)
        assert torch.equal(k_cache[1, page_i, place], k_out[i]) and torch.equal(v_cache[1, page_i, place], v[i])
        k_before[1, page_i, place], v_before[1, page_i, place] = k_out[i], v[i]
    assert torch.equal(k_cache, k_before) and torch.equal(v_cache, v_before)
    cache.append(2, k, v, slots)  # without positions: K as it is
    for i in written:
        page_i, place = divmod(int(slots[i]), page)
        assert torch.equal(k_cache[2, page_i, place], k[i]) and torch.equal(v_cache[2, page_i, place], v[i])
    assert torch.equal(k_cache[:2], k_before[:2])


# ---------------------------------------------------------------- pages
@pytest.mark.parametrize("page,kv_heads,dim", [(8, 1, 64), (16, 3, 128), (256, 8, 128)])
def test_copy_pages(ftg, page, kv_heads, dim):
    gen = _gen(page)
    both = _randn(gen, (2, 3, 2, 20, page, kv_heads, dim), torch.bfloat16)  # layers apart from each other and from V
    k, v = both[0, :, 0], both[1, :, 0]
    cache = ftg.PagedCache(k, v)
    want = both.clone()
    order = torch.randperm(20, generator=gen, device="cuda").to(torch.int32)
    sources, targets = torch.cat([order[:7], order[:2]]), torch.cat([order[7:14], order[14:16]])
    want[:, :, 0, targets.long()] = want[:, :, 0, sources.long()]
    bad = torch.tensor([-1, 20, 3, int(order[0])], dtype=torch.int32, device="cuda")
    cache.copy_pages(torch.cat([sources, bad]), torch.cat([targets, torch.tensor([2, 2, -7, 2 ** 31 - 1], dtype=torch.int32, device="cuda")]))
    assert torch.equal(both, want)
    cache.copy_pages(sources[:0], targets[:0])
    assert torch.equal(both, want)


@pytest.mark.parametrize("page,kv_heads,dim,by_head", [(16, 2, 64, False), (8, 8, 128, False), (64, 5, 128, True), (32, 40, 128, False)])
def test_accept(ftg, page, kv_heads, dim, by_head):
    rng, gen = np.random.RandomState(page), _gen(page)
    contexts, drafted = [0, 5, 100, 63, 40, 7, 9], [4, 30, 1, 150, 8, 6, 0]
    lengths = [c + n for c, n in zip(contexts, drafted)]
    pages, table = _paged(rng, lengths, page)
    shape = (2, pages, kv_heads, page, dim) if by_head else (2, pages, page, kv_heads, dim)
    k, v = _randn(gen, shape, torch.float16), _randn(gen, shape, torch.float16)
    if by_head:
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    paths = [sorted(rng.choice(n, rng.randint(0, n + 1), replace=False)) if n else [] for n in drafted]
    paths[3], paths[4], paths[2] = list(range(20, 150)), list(range(8)), []  # a long overlapping one, all of them, none
    want = [k.clone(), v.clone()]
    for b, path in enumerate(paths):
        for x, old in zip(want, (k, v)):
            for i, node in enumerate(path):
                s, t = contexts[b] + int(node), contexts[b] + i
                x[:, table[b, t // page], t % page] = old[:, table[b, s // page], s % page]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    new, held = ints([7] * 7), ints(lengths)
    ftg.PagedCache(k, v).accept(torch.from_numpy(table).cuda(), held, _offsets(drafted), ints([int(x) for p in paths for x in p]),
                                _offsets([len(p) for p in paths]), new)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    assert new.tolist() == [c + len(p) for c, p in zip(contexts, paths)] and held.tolist() == lengths


def test_accept_leaves_out_what_is_not_there(ftg):
    gen = _gen(1)
    k, v = _randn(gen, (1, 4, 8, 1, 64), torch.float16), _randn(gen, (1, 4, 8, 1, 64), torch.float16)
    before = k.clone(), v.clone()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cache, new = ftg.PagedCache(k, v), ints([0, 0])
    # nodes that were not drafted, and pages outside the cache
    cache.accept(ints([[0, 1], [-1, 9]]), ints([10, 12]), ints([0, 3, 9]), ints([-1, 3, 77, 1, 2]), ints([0, 3, 5]), new)
    assert torch.equal(k, before[0]) and torch.equal(v, before[1]) and new.tolist() == [10, 8]


# ---------------------------------------------------------------- streams, graphs, refusals, and all of it together
def test_streams_and_graphs(ftg):
    gen, dtype = _gen(12), torch.bfloat16
    lengths = [300, 41, 800]
    q, k, v = (_randn(gen, (sum(lengths), h, 128), dtype) for h in (8, 2, 2))
    offsets, out, again = _offsets(lengths), torch.empty_like(q), torch.empty_like(q)
    op = ftg.PromptAttention(8, 2, 128, dtype=dtype)
    op.run(q, k, v, out, offsets)
    k_cache, v_cache = _randn(gen, (1, 40, 64, 2, 128), dtype), _randn(gen, (1, 40, 64, 2, 128), dtype)
    cache = ftg.PagedCache(k_cache, v_cache)
    tree, q1 = ftg.TreeAttention(8, cache), _randn(gen, (3, 8, 128), dtype)
    table = torch.randperm(40, generator=gen, device="cuda")[:39].to(torch.int32).view(3, 13)
    held, out1, again1 = torch.tensor([800, 3, 500], dtype=torch.int32, device="cuda"), torch.empty_like(q1), torch.empty_like(q1)
    tree.run(q1, 0, _offsets([1, 1, 1]), table, held, out1)
    torch.cuda.synchronize()
    # the same inputs give the same bits, on other streams and at the same time as well
    side = [torch.cuda.Stream() for _ in range(2)]
    one_each = _offsets([1, 1, 1])
    torch.cuda.synchronize()
    for _ in range(20):
        op.run(q, k, v, again, offsets, stream=side[0])
        tree.run(q1, 0, one_each, table, held, again1, stream=side[1])
    torch.cuda.synchronize()
    assert torch.equal(out, again) and torch.equal(out1, again1)
    # two graphs, replayed side by side, with lengths that changed since the capture
    graphs = []
    for i, call in enumerate((lambda: op.run(q, k, v, again, offsets), lambda: tree.run(q1, 0, one_each, table, held, again1))):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side[i]):
            call()
        graphs.append(graph)
    held.copy_(torch.tensor([17, 800, 64]))
    tree.run(q1, 0, one_each, table, held, out1)
    again.zero_(), again1.zero_()
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, stream in zip(graphs, side):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, again) and torch.equal(out1, again1)
    op.report(), tree.report()


def test_a_call_with_more_tiles_than_it_can_number_is_refused(ftg):
    """2^10 sequences of up to 2^24 keys with 32 key heads: refused before anything is launched."""
    dtype = torch.bfloat16
    cache = ftg.PagedCache.empty(1, 2, 256, 32, 64, dtype)
    op, batch = ftg.TreeAttention(32, cache), 1 << 10
    q = torch.zeros((batch, 32, 64), dtype=dtype, device="cuda")
    table = torch.zeros((batch, 1 << 16), dtype=torch.int32, device="cuda")
    held = torch.zeros(batch, dtype=torch.int32, device="cuda")
    with pytest.raises(ftg.FtGemmError, match="too large"):
        op.run(q, 0, torch.arange(batch + 1, dtype=torch.int32, device="cuda"), table, held, torch.empty_like(q))


def test_a_captured_step_with_a_padded_batch(ftg):
    """One decoding step of up to six sequences as a graph, replayed with fewer: the sequences that are not there have length
    zero, no queries and negative slots.  Nothing of theirs is written, and the step's launches follow each other in the graph."""
    gen, dtype, page, heads, kv_heads, d = _gen(30), torch.float16, 16, 6, 2, 128
    cache = ftg.PagedCache.empty(2, 30, page, kv_heads, d, dtype)
    cache.k.copy_(_randn(gen, cache.k.shape, dtype)), cache.v.copy_(_randn(gen, cache.v.shape, dtype))
    rotary, tree = ftg.Rotary(d, rotary_dim=64), ftg.TreeAttention(heads, cache)
    q, k, v = (_randn(gen, (6, h, d), dtype) for h in (heads, kv_heads, kv_heads))
    q_out, out = torch.empty_like(q), torch.empty_like(q)
    slots, positions = torch.full((6,), -1, device="cuda"), torch.zeros(6, dtype=torch.int64, device="cuda")
    table = torch.full((6, 5), -1, dtype=torch.int32, device="cuda")
    held, offsets = torch.zeros(6, dtype=torch.int32, device="cuda"), torch.zeros(7, dtype=torch.int32, device="cuda")

    def step():
        cache.append(1, k, v, slots, rotary=rotary, positions=positions, q=q, q_out=q_out)
        tree.run(q_out, 1, offsets, table, held, out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    pages = torch.randperm(30, generator=gen, device="cuda").to(torch.int32).view(6, 5).cpu()
    for real in (6, 2, 0, 5):
        lengths = [int(x) for x in np.random.RandomState(real).randint(1, 80, real)]
        k.copy_(_randn(gen, k.shape, dtype)), v.copy_(_randn(gen, v.shape, dtype)), q.copy_(_randn(gen, q.shape, dtype))
        k[real:], v[real:], q[real:] = math.nan, math.nan, math.nan
        table.fill_(-1), slots.fill_(-1), positions.zero_(), held.zero_(), out.fill_(7.0)
        for i, n in enumerate(lengths):
            table[i] = pages[i]
            slots[i] = int(pages[i, (n - 1) // page]) * page + (n - 1) % page
            positions[i] = n - 1
        held[:real] = torch.tensor(lengths, dtype=torch.int32)
        offsets.copy_(torch.arange(7).clamp(max=real))
        before = [x.clone() for x in (cache.k, cache.v)]
        graph.replay()
        tree.report()
        turned = torch.empty_like(q), torch.empty_like(k)
        rotary.run(q, k, positions, turned[0], turned[1])
        for b, n in enumerate(lengths):
            place = int(slots[b]) // page, int(slots[b]) % page
            before[0][1, place[0], place[1]], before[1][1, place[0], place[1]] = turned[1][b], v[b]
            kk, vv = (x[1, table[b].long()].reshape(-1, kv_heads, d)[:n] for x in before)
            _check_rows(out[b:b + 1], None, turned[0][b:b + 1], kk, vv, torch.ones(1, n, dtype=torch.bool, device="cuda"), d ** -0.5)
        assert torch.equal(before[0], cache.k) and torch.equal(before[1], cache.v)
        assert bool((out[real:] == 7.0).all())


def test_views_of_masks_and_tables(ftg):
    """Rows of masks, page tables and lse of a wider buffer; masks with fewer bits than there are drafted tokens; two rows of the
    table that name the same pages."""
    gen, dtype, page, n, m = _gen(31), torch.bfloat16, 32, 40, 100
    cache = ftg.PagedCache.empty(1, 8, page, 2, 64, dtype)
    cache.k.copy_(_randn(gen, cache.k.shape, dtype)), cache.v.copy_(_randn(gen, cache.v.shape, dtype))
    q = _randn(gen, (2 * n, 8, 64), dtype)
    wide = torch.randint(-2 ** 31, 2 ** 31, (2 * n, 5), generator=gen, device="cuda").to(torch.int32)
    tables = torch.tensor([[7, 5, 0, 3, 9, 9], [7, 5, 0, 3, 9, 9]], dtype=torch.int32, device="cuda")
    out, op = torch.empty_like(q), ftg.TreeAttention(8, cache)
    op.run(q, 0, _offsets([n, n]), tables[:, :4], torch.tensor([m, m], dtype=torch.int32, device="cuda"), out, mask=wide[:, 2:3])
    op.report()
    kk, vv = (x[0, tables[0, :4].long()].reshape(-1, 2, 64)[:m] for x in (cache.k, cache.v))
    bits = (wide[:, 2:3] >> torch.arange(32, device="cuda")) & 1 == 1
    for b in range(2):
        rows = slice(b * n, b * n + n)
        visible = torch.zeros((n, m), dtype=torch.bool, device="cuda")
        visible[:, :m - n] = True
        visible[:, m - n:m - n + 32] = bits[rows]  # the tokens behind the mask's 32 bits are seen by nobody
        _check_rows(out[rows], None, q[rows], kk, vv, visible, 0.125)


def test_keys_that_are_masked_may_hold_anything_in_k(ftg):
    """NaN and infinities in K where a row does not see them, though other rows of the tile do."""
    gen, dtype, n = _gen(32), torch.bfloat16, 150
    q, k, v = (_randn(gen, (n, h, 64), dtype) for h in (4, 1, 1))
    k[100], k[140] = math.nan, math.inf
    out, op = torch.empty_like(q), ftg.PromptAttention(4, 1, 64, dtype=dtype)
    op.run(q, k, v, out, _offsets([n]))
    op.report()
    clean = torch.where(k.isfinite(), k, torch.zeros_like(k))
    _check_rows(out[:100], None, q[:100], clean, v, torch.ones(100, n, dtype=torch.bool, device="cuda").tril(), 0.125)
    assert bool(out[100:].isnan().all())


@pytest.mark.parametrize("page", [8, 16, 64, 256])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("by_head", [False, True])
def test_pages_of_k_and_v_in_turn(ftg, page, dim, by_head):
    """K and V of a page side by side in one buffer, the last page used, the one behind it named."""
    gen, dtype, heads, pages, m = _gen(36), torch.bfloat16, 3, 9, 7 * page + 5
    both = torch.full((2, pages, 2) + ((heads, page, dim) if by_head else (page, heads, dim)), math.nan, dtype=dtype, device="cuda")
    k, v = (both[:, :, i].transpose(2, 3) if by_head else both[:, :, i] for i in range(2))
    cache = ftg.PagedCache(k, v)
    order = [8, 0, 3, 7, 1, 6, 2, 5]
    plain = [_randn(gen, (m, heads, dim), dtype) for _ in range(2)]
    cache.append(1, *plain, torch.tensor([order[i // page] * page + i % page for i in range(m)], device="cuda"))
    q = _randn(gen, (3, 2 * heads, dim), dtype)
    out, op = torch.empty_like(q), ftg.TreeAttention(2 * heads, cache)
    op.run(q, 1, _offsets([3]), torch.tensor([order + [pages]], dtype=torch.int32, device="cuda"), torch.tensor([m], dtype=torch.int32, device="cuda"), out)
    op.report()
    visible = torch.arange(m, device="cuda")[None] <= torch.arange(3, device="cuda")[:, None] + m - 3
    _check_rows(out, None, q, *plain, visible, dim ** -0.5)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("spread", [1.0, 12.0])
def test_pairs_of_row_tiles(ftg, dim, dtype, spread):
    """Enough rows and keys for two row tiles at a time, with scores close together and hundreds apart."""
    gen, lengths, dtype = _gen(34), [1500, 3, 700, 257], DTYPES[dtype]
    q, k, v = (_randn(gen, (sum(lengths), h, dim), dtype, s) for h, s in ((16, spread), (4, spread), (4, 1.0)))
    for causal in (True, False):
        out, lse = torch.empty_like(q), torch.empty((len(q), 16), device="cuda")
        op = ftg.PromptAttention(16, 4, dim, dtype=dtype, causal=causal)
        op.run(q, k, v, out, _offsets(lengths), lse=lse)
        op.report()
        at = 0
        for n in lengths:
            rows, visible = slice(at, at + n), torch.ones(n, n, dtype=torch.bool, device="cuda")
            _check_rows(out[rows], lse[rows], q[rows], k[rows], v[rows], visible.tril() if causal else visible, dim ** -0.5)
            at += n


@pytest.mark.parametrize("dim", [64, 128])
def test_a_nan_in_any_place_of_k_is_seen_by_the_rows_behind_it_only(ftg, dim):
    """64 sequences with a NaN each, every place within 64 keys among them."""
    gen, n, dtype = _gen(35), 400, torch.bfloat16
    q, k, v = (_randn(gen, (64 * n, h, dim), dtype) for h in (4, 1, 1))
    op, offsets, clean, out = ftg.PromptAttention(4, 1, dim, dtype=dtype), _offsets([n] * 64), torch.empty_like(q), torch.empty_like(q)
    op.run(q, k, v, clean, offsets)
    for j in range(64):
        k[j * n + 300 + j] = math.nan
    op.run(q, k, v, out, offsets)
    op.report()
    for j in range(64):
        first = j * n + 300 + j
        assert torch.equal(out[j * n:first], clean[j * n:first]) and bool(out[first:(j + 1) * n].isnan().all()), j


def _climbing(gen, lengths, heads, kv_heads, dim, dtype):
    """Queries of different sizes along one direction and, for each length, keys along it that grow from tile to tile: the
    maxima of the rows rise by 2 to 14 powers of two with every 128 keys."""
    t, keys = sum(n for n, _ in lengths), torch.cat([torch.arange(m, device="cuda") // 128 for _, m in lengths])
    side = torch.randint(0, 2, (dim,), generator=gen, device="cuda") * 2.0 - 1.0
    size = torch.rand((t, heads, 1), generator=gen, device="cuda") + 0.2
    q = (side * size * (64 / dim) ** 0.5 + 0.1 * torch.randn((t, heads, dim), generator=gen, device="cuda")).to(dtype)
    k = (side * keys[:, None, None] + 0.5 * torch.randn((len(keys), kv_heads, dim), generator=gen, device="cuda")).to(dtype)
    return q, k, _randn(gen, (len(keys), kv_heads, dim), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", ["pairs", "split"])
@pytest.mark.parametrize("paged", [False, True])
def test_maxima_that_climb_from_tile_to_tile(ftg, paged, rows, dim, dtype):
    """The accumulator is rescaled at nearly every tile, in both forms: right, and the same bits from run to run."""
    gen, dtype, heads, kv_heads, page = _gen(40), DTYPES[dtype], 8, 2, 64
    lengths = [(1, 2600 - 37 * i) for i in range(40)] if rows == "split" else [(260, 2500), (190, 1800), (500, 2100)]
    q, k, v = _climbing(gen, lengths, heads, kv_heads, dim, dtype)
    offsets, key_offsets = _offsets([n for n, _ in lengths]), _offsets([m for _, m in lengths])
    out, again = torch.empty_like(q), torch.empty_like(q)
    if paged:
        held = [m for _, m in lengths]
        pages, table = _paged(np.random.RandomState(40), held, page)
        cache = ftg.PagedCache.empty(1, pages, page, kv_heads, dim, dtype)
        cache.append(0, k, v, torch.tensor([int(table[b, i // page]) * page + i % page for b, m in enumerate(held) for i in range(m)], device="cuda"))
        op = ftg.TreeAttention(heads, cache)
        args = 0, offsets, torch.from_numpy(table).cuda(), torch.tensor(held, dtype=torch.int32, device="cuda")
        run = lambda to: op.run(q, *args, to)  # noqa: E731
    else:
        op = ftg.PromptAttention(heads, kv_heads, dim, dtype=dtype)
        run = lambda to: op.run(q, k, v, to, offsets, key_offsets=key_offsets)  # noqa: E731
    run(out)
    for _ in range(50):
        run(again)
        assert torch.equal(out, again)
    op.report()
    a = b = 0
    for n, m in lengths:
        visible = torch.arange(m, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] + (m - n)
        _check_rows(out[a:a + n], None, q[a:a + n], k[b:b + m], v[b:b + m], visible, dim ** -0.5)
        a, b = a + n, b + m


@pytest.mark.parametrize("strides", [(640, 128, 3), (128, 1280, 3), (1024, 384, 2), (384, 1024, 3)])
def test_outputs_in_any_layout_whose_rows_are_apart(ftg, strides):
    """By token, by head, and with tokens and heads between each other; broadcast inputs."""
    token, head, heads = strides
    gen, dtype, n, d = _gen(41), torch.bfloat16, 2 if (token, head) == (1024, 384) else 7, 128
    room = torch.full(((n - 1) * token + (heads - 1) * head + d,), 7.0, dtype=dtype, device="cuda")
    out, want = room.as_strided((n, heads, d), (token, head, 1)), torch.empty((n, heads, d), dtype=dtype, device="cuda")
    one, positions = _randn(gen, (n, 1, d), dtype).expand(n, heads, d), torch.arange(n, device="cuda") * 77
    rotary = ftg.Rotary(d)
    rotary.run(one, None, positions, want)
    rotary.run(one, None, positions, out)
    assert torch.equal(out, want) and int((room != 7.0).sum()) <= out.numel()
    with pytest.raises(ftg.FtGemmError, match="share memory"):
        rotary.run(one, None, positions, one)
    q, k = _randn(gen, (n, heads, d), dtype), _randn(gen, (n, 1, d), dtype)
    op = ftg.PromptAttention(heads, 1, d, dtype=dtype)
    op.run(q, k, k, want, _offsets([n]))
    op.run(q, k, k, out, _offsets([n]))
    op.report()
    assert torch.equal(out, want)


def test_masks_written_just_in_front_of_the_call(ftg):
    """The mask changes from call to call, written by the kernel in front on the same stream, in a graph as well."""
    gen, dtype, page, n, m = _gen(42), torch.bfloat16, 32, 60, 200
    cache = ftg.PagedCache.empty(1, 8, page, 2, 64, dtype)
    cache.k.copy_(_randn(gen, cache.k.shape, dtype)), cache.v.copy_(_randn(gen, cache.v.shape, dtype))
    q, out, op = _randn(gen, (n, 8, 64), dtype), torch.empty((n, 8, 64), dtype=dtype, device="cuda"), ftg.TreeAttention(8, cache)
    args = 0, _offsets([n]), torch.arange(7, dtype=torch.int32, device="cuda")[None], torch.tensor([m], dtype=torch.int32, device="cuda")
    masks = torch.randint(-2 ** 31, 2 ** 31, (6, n, 2), generator=gen, device="cuda").to(torch.int32)
    want = []
    for one in masks:
        op.run(q, *args, out, mask=one)
        torch.cuda.synchronize()
        want.append(out.clone())
    assert not any(torch.equal(a, b) for a, b in zip(want, want[1:]))
    mask, got = torch.zeros_like(masks[0]), torch.empty((6, *out.shape), dtype=dtype, device="cuda")

    def calls():
        for i in range(6):
            mask.copy_(masks[i])
            op.run(q, *args, got[i], mask=mask)

    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for replay in range(20):
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        got.zero_(), mask.zero_()
        graph.replay() if replay % 2 else calls()
    op.report()


def test_many_short_prompts_in_a_large_buffer(ftg):
    """All tiles of rows times all keys pass 2^31, what the sequences really have is a small part of it: counted on the device."""
    gen, dtype, batch, heads, d = _gen(43), torch.bfloat16, (1 << 17) + 5, 8, 64
    rng = np.random.RandomState(43)
    counts, key_counts = np.zeros(batch, dtype=np.int64), np.zeros(batch, dtype=np.int64)
    some = sorted(rng.choice(batch, 40, replace=False))
    counts[some], key_counts[some] = rng.randint(1, 200, 40), rng.randint(1, 500, 40)
    tokens, keys = int(counts.sum()), 270_000
    assert (tokens // 128 + batch) * heads * (keys // 128 + 8) > 2 ** 31
    q, k, v = (_randn(gen, (n, heads, d), dtype) for n in (tokens + 3, keys, keys))
    out = torch.full_like(q, 7.0)
    op = ftg.PromptAttention(heads, heads, d, dtype=dtype)
    offsets, key_offsets = _offsets(counts), _offsets(key_counts)
    for _ in range(2):
        op.run(q, k, v, out, offsets, key_offsets=key_offsets)
    op.report()
    a = b = 0
    for n, m in zip(counts[some], key_counts[some]):
        visible = torch.arange(m, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] + (int(m) - int(n))
        _check_rows(out[a:a + n], None, q[a:a + n], k[b:b + m], v[b:b + m], visible, d ** -0.5)
        a, b = a + n, b + m
    assert bool((out[tokens:] == 7.0).all())


def test_packed_prompts_of_too_many_tiles_say_so_and_write_nothing(ftg):
    dtype, heads, n, m = torch.bfloat16, 128, 34_000, 1 << 24
    assert (n // 2) * (m // 128) > 2 ** 31  # 2 tiles of one token's heads at a time
    q, k = torch.zeros((n + 1, heads, 64), dtype=dtype, device="cuda"), torch.zeros((m + 1, 1, 64), dtype=dtype, device="cuda")
    out = torch.full_like(q, 7.0)
    op = ftg.PromptAttention(heads, 1, 64, dtype=dtype)
    op.run(q, k, k, out, _offsets([n, 1]), key_offsets=_offsets([m, 1]))
    with pytest.raises(ftg.FtGemmError, match="too many tiles"):
        op.report()
    assert bool((out == 7.0).all())
    with pytest.raises(ftg.FtGemmError, match="too large"):  # one sequence: known before the launch
        op.run(q, k, k, out, _offsets([n]), key_offsets=_offsets([m]))


def _same_page_over_and_over(ftg, dim, keys, queries):
    """A chain of `queries` zeros over `keys` tokens that all lie in one page, V all ones: (out, lse, how many keys each row sees)."""
    dtype, page = torch.bfloat16, 256
    cache = ftg.PagedCache.empty(1, 1, page, 1, dim, dtype)
    cache.k.fill_(0.5), cache.v.fill_(1.0)
    q = torch.zeros((queries, 1, dim), dtype=dtype, device="cuda")
    out, lse = torch.full_like(q, 7.0), torch.empty((queries, 1), device="cuda")
    table = torch.zeros((1, -(-keys // page)), dtype=torch.int32, device="cuda")
    op = ftg.TreeAttention(1, cache)
    op.run(q, 0, _offsets([queries]), table, torch.tensor([keys], dtype=torch.int32, device="cuda"), out, lse=lse)
    op.report()
    return out, lse, torch.arange(keys - queries + 1, keys + 1, device="cuda")


def test_the_sum_of_very_many_equal_probabilities(ftg):
    """2^26 keys of probability one for every CTA: counts of 64 and their multiples, exact in 32 bits, but ones added to a sum of 2^24
    and more are lost one by one.  The logarithm: a few roundings of a number of its size."""
    rows = 256 * torch.cuda.get_device_properties(0).multi_processor_count
    out, lse, seen = _same_page_over_and_over(ftg, 64, 1 << 26, rows)
    assert bool((out == 1.0).all()), out.float().max().item()
    want = seen.double().log()[:, None]
    assert bool(((lse.double() - want).abs() <= 2.0 ** -21 * (1 + want)).all())


def _repeated_pages(ftg, gen, dim, dtype, lengths, queries, pages, order, heads=2, climb=0.0):
    """Chains over caches whose page table names a few pages of 256 tokens many times: sequence b has the pages order(b), repeated
    as they stand, up to lengths[b].  Checks out and lse in 64 bits by counting how often each row sees each token of a page."""
    page = 256
    cache = ftg.PagedCache.empty(1, pages, page, 1, dim, dtype)
    side = torch.randint(0, 2, (dim,), generator=gen, device="cuda") * 2.0 - 1.0
    q = (side * (torch.rand((sum(queries), heads, 1), generator=gen, device="cuda") + 0.2) * (64 / dim) ** 0.5).to(dtype)
    step = torch.arange(pages, device="cuda")[:, None, None, None] * climb
    cache.k[0].copy_(side * step + torch.randn(cache.k[0].shape, generator=gen, device="cuda"))
    cache.v.copy_(torch.rand(cache.v.shape, generator=gen, device="cuda") + 0.5)  # no two signs: nothing cancels
    width = -(-max(lengths) // page)
    table = torch.stack([order(b, width) for b in range(len(lengths))]).to(torch.int32)
    out, lse, op = torch.full_like(q, 7.0), torch.empty((len(q), heads), device="cuda"), ftg.TreeAttention(heads, cache)
    op.run(q, 0, _offsets(queries), table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), out, lse=lse)
    op.report()
    kd, vd = cache.k[0].double().reshape(-1, dim), cache.v[0].double().reshape(-1, dim)
    u, at = _half_eps(dtype), 0
    for b, (m, n) in enumerate(zip(lengths, queries)):
        seen = torch.arange(m - n + 1, m + 1)  # per row
        whole, rest = seen // page, seen % page
        times = torch.zeros((n, pages), dtype=torch.int64)
        first = int(whole[0])
        times += torch.bincount(table[b, :first].long(), minlength=pages)
        for j in range(first, int(whole[-1])):  # pages that only the later rows see in full
            times[:, int(table[b, j])] += (whole > j).long()
        count = times[:, :, None].expand(n, pages, page).clone()
        last = table[b].long()[whole.clamp(max=width - 1)]
        count[torch.arange(n), last] += (torch.arange(page)[None] < rest[:, None]).long()
        count = count.reshape(n, -1).cuda().double()
        for h in range(heads):
            rows = slice(at, at + n)
            x = (q[rows, h].double() @ kd.T) * dim ** -0.5
            size = ((q[rows, h].double().abs() @ kd.abs().T) * dim ** -0.5).max().item()
            top = x.masked_fill(count == 0, -math.inf).amax(-1, keepdim=True)
            e = count * torch.exp(x - top)
            total = e.sum(-1, keepdim=True)
            want = e @ vd / total  # also the weighted mean of |v|
            s = (dim + 8) * 2.0 ** -24 * max(size, 1.0)
            bound = 1.02 * (2 * u + 2 * s + 2.0 ** -10 + 2.0 ** -13) * want + max(lengths) * 2.0 ** -32 * 1.5
            off = (out[rows, h].double() - want).abs()
            assert bool((off <= bound).all()), f"sequence {b}: off by {(off / want).max().item()}, {(off / bound).max().item()} of the bound"
            want = (top + torch.log(total))[:, 0]
            assert bool(((lse[rows, h].double() - want).abs() <= s + 2.0 ** -13 + 2.0 ** -21 * (1 + want.abs())).all())
        at += n


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", ["pairs", "split"])
@pytest.mark.parametrize("climb", [0.0, 0.6])
def test_millions_of_keys(ftg, dim, dtype, rows, climb):
    """More key tiles of one row tile on one CTA than a side adds up at once (1024, 2^17 keys: at most N 2^-27 = 2^-10 of the sum is cut off;
    2 x 1024 further additions, 2^-13); page after page of larger scores when they climb, so that what is kept shrinks."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    pages = 8
    in_turn = lambda b, width: torch.arange(width) * pages // width if climb else (torch.arange(width) + b) % pages  # noqa: E731
    if rows == "pairs":
        _repeated_pages(ftg, _gen(45), dim, DTYPES[dtype], [600_001, 2_000_123], [64 * sms + 77, 64 * sms], pages, in_turn, climb=climb)
    else:
        lengths = [1_000_001 + 9973 * b for b in range(60)]
        _repeated_pages(ftg, _gen(46), dim, DTYPES[dtype], lengths, [1] * 60, pages, in_turn, climb=climb)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", ["pairs", "split"])
def test_millions_of_packed_keys(ftg, dim, dtype, rows):
    """The same over packed keys, growing towards the end; some of the rows are checked."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    gen, dtype, heads = _gen(47), DTYPES[dtype], 2
    n, m = (128 * sms, 300_001) if rows == "pairs" else (1, 2 * 1200 * 128 * sms + 77)
    side = torch.randint(0, 2, (dim,), generator=gen, device="cuda") * 2.0 - 1.0
    q = (side * (torch.rand((n, heads, 1), generator=gen, device="cuda") + 0.2) * (64 / dim) ** 0.5).to(dtype)
    k, v = torch.empty((m, 1, dim), dtype=dtype, device="cuda"), torch.empty((m, 1, dim), dtype=dtype, device="cuda")
    pieces = [(a, min(a + (1 << 20), m)) for a in range(0, m, 1 << 20)]
    for a, b in pieces:
        grow = torch.arange(a, b, device="cuda")[:, None, None] * (4.0 / m)
        k[a:b] = side * grow + torch.randn((b - a, 1, dim), generator=gen, device="cuda")
        v[a:b] = torch.rand((b - a, 1, dim), generator=gen, device="cuda") + 0.5
    out, lse, op = torch.full_like(q, 7.0), torch.empty((n, heads), device="cuda"), ftg.PromptAttention(heads, 1, dim, dtype=dtype)
    op.run(q, k, v, out, _offsets([n]), key_offsets=_offsets([m]), lse=lse)
    op.report()
    some = torch.tensor(sorted({0, n // 3, n // 2, n - 1}), device="cuda")
    x = [(q[some].double().reshape(-1, dim) @ k[a:b, 0].double().T) * dim ** -0.5 for a, b in pieces]
    sees = (some + m - n).repeat_interleave(heads)[:, None]  # the last key of each row
    x = torch.cat(x, 1).masked_fill(torch.arange(m, device="cuda")[None] > sees, -math.inf)
    size = x.masked_fill(x == -math.inf, 0.0).abs().max().item() + 8.0 * dim ** 0.5  # of the sum of magnitudes: |q| |k| is at most some units more
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    want = sum(e[:, a:b] @ v[a:b, 0].double() for a, b in pieces) / total
    u, s = _half_eps(dtype), (dim + 8) * 2.0 ** -24 * size
    bound = 1.02 * (2 * u + 2 * s + 2.0 ** -10 + 2.0 ** -13) * want + m * 2.0 ** -32 * 1.5
    off = (out[some].double().reshape(-1, dim) - want).abs()
    assert bool((off <= bound).all()), f"off by {(off / want).max().item()}, {(off / bound).max().item()} of the bound"
    want = (top + torch.log(total))[:, 0]
    assert bool(((lse[some].double().reshape(-1) - want).abs() <= s + 2.0 ** -13 + 2.0 ** -21 * (1 + want.abs())).all())


def test_a_row_tile_over_as_many_keys_as_there_can_be(ftg):
    """2^27 keys in one item per CTA (seconds of work): the warp that clears the rows behind the last key waits for all of it.  The sums:
    multiples of 64 up to 2^26 for each half of the keys, then one addition."""
    keys, rows = (1 << 27) - 5, 256 * torch.cuda.get_device_properties(0).multi_processor_count
    out, lse, seen = _same_page_over_and_over(ftg, 128, keys, rows)
    assert bool((out == 1.0).all()), (out.float().min().item(), out.float().max().item())
    want = seen.double().log()[:, None]
    assert bool(((lse.double() - want).abs() <= 2.0 ** -21 * (1 + want)).all())


def test_a_call_waits_for_what_another_stream_has_written(ftg):
    """Its kernels may begin while the one in front on their stream runs, but not in front of an event that the stream waits for:
    keys appended and queries made on a side stream that is late, eagerly and in a graph with a fork and a join."""
    gen, dtype, page, heads, kv_heads, d = _gen(44), torch.bfloat16, 16, 8, 2, 64
    cache = ftg.PagedCache.empty(1, 64, page, kv_heads, d, dtype)
    slow = _randn(gen, (4096, 4096), dtype)
    lengths = [300, 17, 500]
    source = [_randn(gen, (sum(lengths), h, d), dtype) for h in (heads, kv_heads, kv_heads)]
    q, out = torch.empty_like(source[0]), torch.empty_like(source[0])
    pages, table = _paged(np.random.RandomState(44), lengths, page, spare=0)
    slots = torch.tensor([int(table[b, i // page]) * page + i % page for b, n in enumerate(lengths) for i in range(n)], device="cuda")
    offsets, table = _offsets(lengths), torch.from_numpy(table).cuda()
    held, tree, prompt = torch.tensor(lengths, dtype=torch.int32, device="cuda"), ftg.TreeAttention(heads, cache), ftg.PromptAttention(heads, kv_heads, d, dtype=dtype)
    packed, side, main = torch.empty_like(out), torch.cuda.Stream(), torch.cuda.Stream()

    def calls():
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(8):
                torch.mm(slow, slow)
            cache.append(0, source[1], source[2], slots)
            q.copy_(source[0])
        out.zero_(), packed.zero_()  # a short kernel right in front, on this stream
        torch.cuda.current_stream().wait_stream(side)
        tree.run(q, 0, offsets, table, held, out)
        prompt.run(q, source[1], source[2], packed, offsets)

    def clear():
        torch.cuda.synchronize()
        q.fill_(math.nan), cache.k.fill_(math.nan), cache.v.fill_(math.nan)
        torch.cuda.synchronize()

    graph = None
    for turn in range(6):
        clear()
        with torch.cuda.stream(main):
            if turn < 3:
                calls()
            elif graph is None:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=main):
                    calls()
                graph.replay()
            else:
                graph.replay()
        tree.report(), prompt.report()
        at = 0
        for n in lengths:
            rows, visible = slice(at, at + n), torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
            for got in (out, packed):
                _check_rows(got[rows], None, source[0][rows], source[1][rows], source[2][rows], visible, d ** -0.5)
            at += n


def test_the_pool_refuses_to_be_captured(ftg):
    """Before anything changes: its copies would be lost, and the pages would be taken for copied."""
    cache = ftg.PagedCache.empty(1, 6, 8, 1, 64)
    cache.k.fill_(1.0), cache.v.fill_(1.0)
    pool = ftg.PagePool(6, 8, cache)
    first, a = pool.new_sequence(), pool.new_sequence()
    pool.extend([first, a], [8, 5])
    b = pool.fork(a)
    pool.free(first)
    before, x = [pool.page_list(s) for s in (a, b)], torch.zeros(4, device="cuda")
    for call in (lambda: pool.extend([a], [1]), lambda: pool.compact()):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            x.add_(1.0)
            with pytest.raises(RuntimeError, match="captured step"):
                call()
        graph.replay()
        assert [pool.page_list(s) for s in (a, b)] == before and pool.length(a) == 5 and pool.free_pages() == 5
    torch.cuda.synchronize()
    assert x.tolist() == [2.0] * 4
    side = torch.cuda.Stream()
    assert pool.extend([a], [1], stream=side) == [(1, 0)] and pool.compact() == []  # otherwise as ever; the copy fills the hole


@pytest.mark.parametrize("code", ["FT_ERR_TIMEOUT", "FT_ERR_INVALID"])
def test_a_reported_failure_does_not_count_against_later_runs(ftg, code):
    """The status word is set here as a kernel would set it."""
    x, op = torch.ones((5, 2, 64), dtype=torch.bfloat16, device="cuda"), ftg.PromptAttention(2, 2, 64)
    op.status.fill_(getattr(ftg, code))
    with pytest.raises(ftg.FtGemmError, match="not valid" if code == "FT_ERR_TIMEOUT" else "wrote nothing"):
        op.report()
    out = torch.empty_like(x)
    op.run(x, x, x, out, _offsets([5]))
    op.report()
    assert bool((out == 1.0).all())


def test_page_operations_and_rotary_positions_in_graphs_and_on_streams(ftg):
    gen, dtype = _gen(33), torch.bfloat16
    cache = ftg.PagedCache.empty(2, 12, 8, 2, 64, dtype)
    start = [_randn(gen, cache.k.shape, dtype) for _ in range(2)]
    sources, targets = torch.tensor([3, 1, 3], dtype=torch.int32, device="cuda"), torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 2, 4], [9, 8, 10]], dtype=torch.int32, device="cuda")
    held, drafted = torch.tensor([20, 9], dtype=torch.int32, device="cuda"), _offsets([9, 4])
    accepted, ends, new = torch.tensor([0, 3, 8, 1, 3], dtype=torch.int32, device="cuda"), _offsets([3, 2]), torch.empty(2, dtype=torch.int32, device="cuda")
    rotary, x = ftg.Rotary(64), _randn(gen, (5, 3, 64), dtype)
    positions, twice = torch.arange(5, device="cuda") * 1000, torch.empty_like(x)

    def calls(stream=None):
        cache.copy_pages(sources, targets, stream=stream)
        cache.accept(table, held, drafted, accepted, ends, new, stream=stream)
        rotary.run(x, None, positions, twice, stream=stream)
        rotary.run(twice, None, positions, twice, inverse=True, stream=stream)  # in place

    results = []
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    for way in range(3):
        cache.k.copy_(start[0]), cache.v.copy_(start[1]), new.zero_(), twice.zero_()
        torch.cuda.synchronize()
        if way == 0:
            calls()
        elif way == 1:
            calls(side)
        else:
            with torch.cuda.graph(graph):
                calls()
            assert torch.equal(cache.k, start[0])  # captured only
            graph.replay()
        torch.cuda.synchronize()
        results.append([y.clone() for y in (cache.k, cache.v, new, twice)])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
    want = [y.clone() for y in start]
    for y in want:
        y[:, [5, 6, 7]] = y[:, [3, 1, 3]]
        for b, (n, own, kept) in enumerate(((20, 9, [0, 3, 8]), (9, 4, [1, 3]))):
            flat = lambda i: (int(table[b, i // 8]), i % 8)  # noqa: E731
            rows = [y[:, flat(n - own + j)[0], flat(n - own + j)[1]].clone() for j in kept]
            for i, row in enumerate(rows):
                y[:, flat(n - own + i)[0], flat(n - own + i)[1]] = row
    assert torch.equal(results[0][0], want[0]) and torch.equal(results[0][1], want[1])
    assert results[0][2].tolist() == [14, 7]
    # there and back: two roundings of numbers that a rotation makes at most sqrt(2) times as large, and 2^-24-sized errors
    pair = (x[..., :32].double() ** 2 + x[..., 32:].double() ** 2).sqrt()
    off = (results[0][3].double() - x.double()).abs().amax(-1, keepdim=True)
    bound = 1.02 * (2 * math.sqrt(2) * _half_eps(dtype)) * pair.amax(-1, keepdim=True) + 1e-30
    assert bool((off <= bound).all())


def test_refusals(ftg):
    dtype = torch.bfloat16
    x = torch.zeros((4, 2, 64), dtype=dtype, device="cuda")
    op = ftg.PromptAttention(2, 2, 64, dtype=dtype)
    offsets = _offsets([4])
    for bad in (dict(q=x.float()), dict(q=x[:, :1]), dict(k=x.cpu()), dict(out=x[:3]), dict(v=x.transpose(1, 2)), dict(offsets=offsets.long()),
                dict(offsets=offsets.cpu()), dict(key_offsets=_offsets([2, 2])), dict(lse=x[:, :, 0])):
        with pytest.raises(ValueError):
            op.run(**{**dict(q=x, k=x, v=x, out=x.clone(), offsets=offsets), **bad})
    with pytest.raises(ValueError, match="key_offsets"):
        op.run(x, x[:2], x[:2], x.clone(), offsets)
    wide = torch.zeros((4, 2, 66), dtype=dtype, device="cuda")
    with pytest.raises(ftg.FtGemmError, match="16-byte"):
        op.run(wide[..., :64], x, x, x.clone(), offsets)
    with pytest.raises(ftg.FtGemmError):
        op.run(x, x[:, :1].expand(4, 2, 64), x, x.clone(), offsets)  # heads that share memory
    with pytest.raises(ftg.FtGemmError, match="head_dim"):
        ftg.PromptAttention(2, 2, 32, dtype=dtype).run(x[..., :32].contiguous(), x[..., :32].contiguous(), x[..., :32].contiguous(),
                                                       x[..., :32].contiguous(), offsets)
    with pytest.raises(ftg.FtGemmError, match="times the key heads"):
        ftg.PromptAttention(2, 4, 64, dtype=dtype).run(x, torch.zeros((4, 4, 64), dtype=dtype, device="cuda"), torch.zeros((4, 4, 64), dtype=dtype, device="cuda"),
                                                       x.clone(), offsets)
    cache = ftg.PagedCache.empty(1, 2, 16, 2, 64, dtype)
    with pytest.raises(ftg.FtGemmError, match="page_size"):
        ftg.PagedCache.empty(1, 2, 24, 2, 64, dtype)
    with pytest.raises(ftg.FtGemmError, match="layer"):
        cache.append(1, x, x, torch.zeros(4, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="slots"):
        cache.append(0, x, x, torch.zeros(4, dtype=torch.int32, device="cuda"))
    tree = ftg.TreeAttention(4, cache)
    q, table, held = torch.zeros((4, 4, 64), dtype=dtype, device="cuda"), torch.zeros((1, 2), dtype=torch.int32, device="cuda"), offsets[1:]
    for bad in (dict(page_table=table[:0]), dict(lengths=offsets), dict(mask=table), dict(q=x)):
        with pytest.raises(ValueError):
            tree.run(**{**dict(q=q, layer=0, offsets=offsets, page_table=table, lengths=held, out=q.clone()), **bad})
    with pytest.raises(ftg.FtGemmError, match="layer"):
        tree.run(q, 1, offsets, table, held, q.clone())
    rotary = ftg.Rotary(64)
    with pytest.raises(ValueError):
        rotary.run(x, x, torch.zeros(4, dtype=torch.int32, device="cuda"), x, x)
    with pytest.raises(ValueError, match="together"):
        rotary.run(x, x, torch.zeros(4, dtype=torch.int64, device="cuda"), x)
    # nothing to do is no error
    op.run(x[:0], x[:0], x[:0], x[:0], offsets[:1])
    rotary.run(x[:0], None, torch.zeros(0, dtype=torch.int64, device="cuda"), x[:0])


def test_attention_program_with_rotary_positions_and_without_protection(ftg):
    """The command-line program rotates its inputs and runs the prompt attention beside the protected one; both are verified
    in 64 bits on the same rows."""
    exe = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "build", "ft_flash_attention")
    if not os.path.exists(exe):
        pytest.skip("the command-line programs are not built")
    for extra in (["--causal", "--rotary"], ["--rotary", "--rotary-base", "500000", "--head-dim", "64", "--sequence", "333"], []):
        out = subprocess.run([exe, *extra, "--batch", "2", "--heads", "3", "--sequence", "512", "--repeat", "2", "--verify-rows", "600", "--unprotected"],
                             capture_output=True, text=True, timeout=300)
        report = dict(line.split(": ", 1) for line in out.stdout.splitlines() if ": " in line)
        assert out.returncode == 0 and report["verification"] == "PASS", out.stdout + out.stderr
        assert float(report["unprotected_max_absolute_error"]) < 4e-3 and float(report["unprotected_time_ms"]) > 0
        assert ("rotary_base" in report) == ("--rotary" in extra)


def test_a_served_decoder_step_by_step(ftg):
    """The operators as they are used together: prompts in, a fork, drafted trees, verification, and on; at each point the
    attention over the cache equals the attention over everything the sequence has kept."""
    gen, rng, dtype = _gen(20), np.random.RandomState(20), torch.bfloat16
    heads, kv_heads, d, page, layers = 8, 2, 64, 16, 2
    rotary = ftg.Rotary(d, scaling="by_parts", factor=4.0, original_length=64)
    cache = ftg.PagedCache.empty(layers, 40, page, kv_heads, d, dtype)
    cache.k.fill_(math.nan), cache.v.fill_(math.nan)
    pool = ftg.PagePool(40, page, cache)
    prompt, tree = ftg.PromptAttention(heads, kv_heads, d, dtype=dtype), ftg.TreeAttention(heads, cache)
    kept = {}  # sequence -> per layer [k, v] rows, K rotated

    def rows(tokens):
        return [_randn(gen, (tokens, h, d), dtype) for h in (heads, kv_heads, kv_heads)]

    def append(sequences, positions, counts, first):
        slots = torch.tensor([x for s, n, f in zip(sequences, counts, first) for x in pool.slots(s, f, n)], device="cuda")
        made = []
        for layer in range(layers):
            q, k, v = rows(sum(counts))
            q_out = torch.empty_like(q)
            cache.append(layer, k, v, slots, rotary=rotary, positions=positions, q=q, q_out=q_out)
            k_out = torch.empty_like(k)
            rotary.run(q, k, positions, torch.empty_like(q), k_out)
            made.append((q_out, k_out, v))
        return made

    # two prompts, packed
    lengths = [37, 70]
    sequences = [pool.new_sequence() for _ in lengths]
    pool.extend(sequences, lengths)
    made = append(sequences, torch.cat([torch.arange(n, device="cuda") for n in lengths]), lengths, [0, 0])
    at = 0
    for s, n in zip(sequences, lengths):
        kept[s] = [[k[at:at + n], v[at:at + n]] for _, k, v in made]
        at += n
    for layer, (q, k, v) in enumerate(made):
        a, b = torch.empty_like(q), torch.empty_like(q)
        prompt.run(q, k, v, a, _offsets(lengths))
        table, held = pool.table(sequences)
        tree.run(q, layer, _offsets(lengths), table, held, b)  # the same as a chain over the cache
        at = 0
        for s, n in zip(sequences, lengths):
            for out in (a, b):
                _check_rows(out[at:at + n], None, q[at:at + n], *kept[s][layer], torch.ones(n, n, dtype=torch.bool, device="cuda").tril(), d ** -0.5)
            at += n
    # a fork of the second; then drafted trees for all three, three times over
    child = pool.fork(sequences[1])
    kept[child] = [list(x) for x in kept[sequences[1]]]
    sequences.append(child)
    for turn in range(3):
        counts = [int(rng.randint(1, 12)) for _ in sequences]
        first = [pool.length(s) for s in sequences]
        pool.extend(sequences, counts)
        trees = [[-1] + [int(rng.randint(0, i)) for i in range(1, n)] for n in counts]
        masks = [ftg.tree_mask(p, 1) for p in trees]
        depth = [[bin(int(m) & 0xFFFFFFFF).count("1") - 1 for m in mask[:, 0]] for mask in masks]
        positions = torch.tensor([f + x for f, ds in zip(first, depth) for x in ds], device="cuda")
        made = append(sequences, positions, counts, first)
        table, held = pool.table(sequences)
        packed, offsets = torch.cat(masks).cuda(), _offsets(counts)
        for layer, (q, k, v) in enumerate(made):
            out = torch.empty_like(q)
            tree.run(q, layer, offsets, table, held, out, mask=packed)
            at = 0
            for s, n, f, mask in zip(sequences, counts, first, masks):
                own = (mask >> torch.arange(n)[None]) & 1 == 1
                visible = torch.cat([torch.ones(n, f, dtype=torch.bool), own], 1).cuda()
                kk, vv = (torch.cat([old, new[at:at + n]]) for old, new in zip(kept[s][layer], (k, v)))
                _check_rows(out[at:at + n], None, q[at:at + n], kk, vv, visible, d ** -0.5)
                at += n
        # the path to one node of each tree is accepted
        paths = []
        for n, mask in zip(counts, masks):
            bits = int(mask[rng.randint(0, n), 0]) & 0xFFFFFFFF
            paths.append([j for j in range(n) if bits >> j & 1])
        new = torch.empty_like(held)
        cache.accept(table, held, offsets, torch.tensor([x for p in paths for x in p], dtype=torch.int32, device="cuda"),
                     _offsets([len(p) for p in paths]), new)
        at = 0
        for s, n, f, path in zip(sequences, counts, first, paths):
            for layer, (_, k, v) in enumerate(made):
                pick = torch.tensor([at + x for x in path], device="cuda")
                kept[s][layer] = [torch.cat([kept[s][layer][0], k[pick]]), torch.cat([kept[s][layer][1], v[pick]])]
            pool.truncate(s, f + len(path))
            at += n
        assert new.tolist() == [pool.length(s) for s in sequences]
        if turn == 0:
            pool.free(sequences.pop(0))
            pool.compact()
    table, held = pool.table(sequences)
    for layer in range(layers):
        q = rows(len(sequences))[0]
        out = torch.empty_like(q)
        tree.run(q, layer, _offsets([1] * len(sequences)), table, held, out)
        for i, s in enumerate(sequences):
            kk, vv = kept[s][layer]
            _check_rows(out[i:i + 1], None, q[i:i + 1], kk, vv, torch.ones(1, len(kk), dtype=torch.bool, device="cuda"), d ** -0.5)
    prompt.report(), tree.report()
