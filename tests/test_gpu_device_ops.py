"""The device-pointer operators against plain 64-bit computations, at the sizes and masks where they can go wrong."""
import math
import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(backend):
    from funasrnet_b200.device_ops import DeviceOps

    return DeviceOps(backend)


def torch_():
    import torch

    return torch


def dtype_of(name):
    torch = torch_()
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def here():
    return torch_().cuda.current_stream().cuda_stream


def randn(seed, *shape, dtype):
    torch = torch_()
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def i32(values):
    return torch_().tensor(values, dtype=torch_().int32, device="cuda")


def sums(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).tolist()


def packed_space(dev, q, k, qo):
    return torch_().empty(max(16, dev.attention_packed_workspace(q, k, qo)), dtype=torch_().uint8, device="cuda")


def visible(new, keys, causal):
    torch = torch_()
    i, j = torch.arange(new, device="cuda")[:, None], torch.arange(keys, device="cuda")
    see = torch.ones(new, keys, dtype=torch.bool, device="cuda")
    return see & (j <= i + keys - new) if causal else see


def check_packed(q, k, v, new, keys, causal, scale, out, lse, start=(0, 0)):
    import dev_reference as R

    qo, ko = start
    for b, (n, m) in enumerate(zip(new, keys)):
        if n:
            want = R.attention(q[qo:qo + n], k[ko:ko + m], v[ko:ko + m], scale, visible(n, m, causal), q.dtype)
            R.check(out[qo:qo + n], want[0], want[2], f"sequence {b} out")
            R.check(lse[qo:qo + n], want[1], want[3], f"sequence {b} lse")
        qo, ko = qo + n, ko + m


PACKED = [
    # heads, kv_heads, head_size, queries, keys (None: as queries), causal
    (1, 1, 8, [1], None, True),
    (2, 2, 64, [1, 1, 1], [1, 129, 4000], True),
    (16, 8, 128, [37], None, True),
    (16, 8, 128, [64, 65, 127, 128, 129, 1], None, True),
    (16, 8, 128, [256, 0, 257, 0], None, False),
    (4, 1, 64, [300, 511], [700, 1024], True),
    (12, 4, 96, [85, 86, 43], [85, 300, 129], True),
    (14, 2, 64, [18, 19, 36, 37], None, True),
    (20, 4, 80, [100, 1], [228, 128], False),
    (8, 8, 40, [130], [128], True),          # the first two queries see no key
    (4, 2, 128, [5, 7], [0, 3], True),       # no keys at all; fewer keys than queries
    (64, 1, 128, [3, 2], [130, 64], True),
    (6, 6, 112, [200], [383], True),
    (3, 1, 24, [1000], None, True),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,size,new,keys,causal", PACKED)
def test_packed_matches_64_bits(dev, dtype, heads, kv_heads, size, new, keys, causal):
    torch = torch_()
    keys = new if keys is None else keys
    dt = dtype_of(dtype)
    q, k, v = (randn(1 + i, sum(n), h, size, dtype=dt) for i, (n, h) in enumerate(((new, heads), (keys, kv_heads), (keys, kv_heads))))
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    qo, ko = i32(sums(new)), i32(sums(keys))
    assert dev.attention_packed(q, k, v, qo, ko, out, causal=causal, lse=lse, workspace=packed_space(dev, q, k, qo),
                                stream=here())
    torch.cuda.synchronize()
    check_packed(q, k, v, new, keys, causal, size ** -0.5, out, lse)
    dev.status()


def test_packed_strided_fused_projection_and_rows_behind(dev):
    """q, k and v as slices of one fused projection, head-major output, offsets that start past 0, and rows of no sequence."""
    torch = torch_()
    heads, kv_heads, size, new = 16, 8, 128, [70, 140]
    total = 5 + sum(new) + 9
    qkv = randn(3, total, heads + 2 * kv_heads, size, dtype=torch.float16)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    out = torch.full((heads, total, size), 3.0, dtype=torch.float16, device="cuda").permute(1, 0, 2)
    lse = torch.full((total, heads), 3.0, device="cuda")
    off = i32([5, 75, 215])
    assert dev.attention_packed(q, k, v, off, off, out, scale=0.2, lse=lse, workspace=packed_space(dev, q, k, off),
                                stream=here())
    torch.cuda.synchronize()
    check_packed(q, k, v, new, new, True, 0.2, out, lse, start=(5, 5))
    for t in (out, lse):
        assert (t[:5] == 3.0).all() and (t[215:] == 3.0).all()


def test_packed_values_that_are_not_finite_stay_with_their_sequence(dev):
    """NaN and infinities of one sequence, and of rows that no sequence owns, reach no other sequence."""
    torch = torch_()
    new = [50, 60, 70]
    q, k, v = (randn(4 + i, 200, 4, 64, dtype=torch.bfloat16) for i in range(3))
    k[50:110], v[50:110] = math.nan, math.inf
    k[180:], v[180:] = math.inf, math.nan
    out, lse = torch.zeros_like(q), torch.zeros(200, 4, device="cuda")
    off = i32(sums(new))
    assert dev.attention_packed(q, k, v, off, off, out, causal=False, lse=lse,
                                workspace=packed_space(dev, q, k, off), stream=here())
    torch.cuda.synchronize()
    check_packed(q[:50], k[:50], v[:50], [50], [50], False, 0.125, out[:50], lse[:50])
    check_packed(q[110:180], k[110:180], v[110:180], [70], [70], False, 0.125, out[110:180], lse[110:180])
    assert torch.isnan(out[50:110]).all()


def test_packed_scores_over_a_wide_range(dev):
    """Scores that rise by hundreds along the keys (the running maximum moves at every tile) and -inf scores."""
    torch = torch_()
    n, size = 700, 64
    q = randn(7, n, 2, size, dtype=torch.bfloat16)
    k = randn(8, n, 2, size, dtype=torch.bfloat16) * torch.linspace(0.1, 20, n, device="cuda")[:, None, None].bfloat16()
    v = randn(9, n, 2, size, dtype=torch.bfloat16)
    out, lse = torch.zeros_like(q), torch.zeros(n, 2, device="cuda")
    off = i32([0, n])
    assert dev.attention_packed(q, k, v, off, off, out, scale=1.0, lse=lse, workspace=packed_space(dev, q, k, off),
                                stream=here())
    torch.cuda.synchronize()
    check_packed(q, k, v, [n], [n], True, 1.0, out, lse)


# ------------------------------------------------------------ shared prefix ----


def shared_space(dev, q, pk, sk):
    return torch_().empty(max(16, dev.attention_shared_workspace(q, pk, sk)), dtype=torch_().uint8, device="cuda")


def check_shared(q, pk, pv, sk, sv, lens, scale, out, lse):
    import dev_reference as R

    torch = torch_()
    for b, n in enumerate(lens):
        k, v = torch.cat([pk, sk[b, :n]]), torch.cat([pv, sv[b, :n]])
        see = torch.ones(1, k.shape[0], dtype=torch.bool, device="cuda")
        want = R.attention(q[b:b + 1], k, v, scale, see, q.dtype)
        R.check(out[b:b + 1], want[0], want[2], f"sequence {b} out")
        R.check(lse[b:b + 1], want[1], want[3], f"sequence {b} lse")


SHARED = [
    # heads, kv_heads, head_size, prefix, suffix lengths
    (1, 1, 8, 1, [0]),
    (16, 8, 128, 61, [0, 7]),
    (16, 8, 128, 0, [5, 0, 129, 16]),
    (16, 8, 128, 130, [0, 0, 0]),
    (16, 8, 128, 2049, list(range(0, 70))),
    (32, 4, 64, 1000, [1, 15, 16, 17, 31, 32, 33, 64, 300]),
    (14, 2, 96, 383, [100] * 20 + [3]),
    (20, 4, 80, 128, [77, 0, 200]),
    (64, 1, 128, 300, [40, 41, 42]),
    (6, 6, 40, 5000, [1]),
    (8, 1, 112, 129, list(range(100, 230))),
    (3, 1, 24, 0, [0, 1, 2]),
    (8, 2, 128, 9000, [4000]),
    (32, 4, 64, 5000, [0, 1, 70, 33] * 20),      # large enough together for the tensor cores, in several shapes
    (14, 2, 96, 4003, [5] * 119 + [130]),
    (64, 1, 128, 5001, [64, 65] * 50),
    (6, 6, 40, 1200, [1, 2, 3] * 50),
    (32, 8, 128, 6, list(range(217, 804, 31))),  # keys cut into parts that a cluster joins
    (8, 1, 112, 6403, [47, 48, 0, 47]),          # into more parts than a cluster has
    (16, 16, 64, 130, list(range(0, 240, 4))),   # more rows than the SMs hold at a time
    (12, 6, 48, 3, [1, 0, 77] * 40),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,size,prefix,lens", SHARED)
def test_shared_matches_64_bits(dev, dtype, heads, kv_heads, size, prefix, lens):
    """Cache rows behind a sequence's length hold NaN: they are not used."""
    torch = torch_()
    dt = dtype_of(dtype)
    n, cap = len(lens), max(lens) + 3
    q, out = randn(1, n, heads, size, dtype=dt), torch.full((n, heads, size), 7.0, dtype=dt, device="cuda")
    pk, pv = randn(2, prefix, kv_heads, size, dtype=dt), randn(3, prefix, kv_heads, size, dtype=dt)
    sk, sv = randn(4, n, cap, kv_heads, size, dtype=dt), randn(5, n, cap, kv_heads, size, dtype=dt)
    for b, m in enumerate(lens):
        sk[b, m:], sv[b, m:] = math.nan, math.nan
    lse = torch.full((n, heads), 7.0, device="cuda")
    assert dev.attention_shared(q, pk, pv, sk, sv, i32(lens), out, lse=lse, workspace=shared_space(dev, q, pk, sk),
                                stream=here())
    torch.cuda.synchronize()
    check_shared(q, pk, pv, sk, sv, lens, size ** -0.5, out, lse)
    dev.status()


def test_shared_head_major_cache_and_no_suffix_capacity(dev):
    """The sessions' cache layout [sequence][KV head][position][size], and a suffix of capacity 0."""
    torch = torch_()
    n, heads, kv_heads, size, prefix, cap, lens = 5, 16, 8, 128, 300, 90, [90, 1, 0, 33, 64]
    q, out = randn(1, n, heads, size, dtype=torch.float16), torch.zeros(n, heads, size, dtype=torch.float16, device="cuda")
    pk, pv = (randn(2 + i, kv_heads, prefix, size, dtype=torch.float16).permute(1, 0, 2) for i in range(2))
    sk, sv = (randn(4 + i, n, kv_heads, cap, size, dtype=torch.float16).permute(0, 2, 1, 3) for i in range(2))
    lse = torch.zeros(n, heads, device="cuda")
    assert dev.attention_shared(q, pk, pv, sk, sv, i32(lens), out, lse=lse, workspace=shared_space(dev, q, pk, sk),
                                stream=here())
    torch.cuda.synchronize()
    check_shared(q, pk, pv, sk, sv, lens, size ** -0.5, out, lse)
    none = sk[:, :0]
    assert dev.attention_shared(q, pk, pv, none, none, i32([0] * n), out, lse=lse,
                                workspace=shared_space(dev, q, pk, none), stream=here())
    torch.cuda.synchronize()
    check_shared(q, pk, pv, none, none, [0] * n, size ** -0.5, out, lse)


# ------------------------------------------------------------------- logits ----


def adjust_case(dev, dtype, rows, vocab, seed, history=True, biases=True, masks=True, hist_max=60, in_place=False, pad=0):
    torch = torch_()
    rng = random.Random(seed)
    dt = dtype_of(dtype)
    x = (randn(seed, rows, vocab + pad, dtype=torch.float32) * 3).to(dt)[:, pad // 2:pad // 2 + vocab]
    out = x.clone() if not in_place else x
    x0 = x.clone()
    tokens = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
    kw = {}
    hist = [[rng.choice([rng.randrange(vocab), vocab - 1, 0, -1, vocab]) for _ in range(rng.randint(0, hist_max))] for _ in range(rows)]
    prompt = [rng.randint(0, len(h) + 2) for h in hist]
    rep, pres, freq = ([rng.uniform(*r) for _ in range(rows)] for r in ((0.7, 1.5), (-0.5, 0.9), (-0.2, 0.4)))
    rep, pres, freq = (np.asarray(a, np.float32).astype(np.float64).tolist() for a in (rep, pres, freq))
    if history:
        kw.update(history=i32([t for h in hist for t in h]), history_offsets=i32(sums([len(h) for h in hist])),
                  prompt_lens=i32(prompt), repetition=torch.tensor(rep, device="cuda", dtype=torch.float32),
                  presence=torch.tensor(pres, device="cuda", dtype=torch.float32),
                  frequency=torch.tensor(freq, device="cuda", dtype=torch.float32))
    bias = [[(rng.choice([rng.randrange(vocab), 3 % vocab, -5, vocab + 2]), float(np.float32(rng.uniform(-4, 4))))
             for _ in range(rng.randint(0, 30))] for _ in range(rows)]
    if biases:
        kw.update(bias_tokens=i32([t for b in bias for t, _ in b]),
                  bias_values=torch.tensor([v for b in bias for _, v in b], device="cuda", dtype=torch.float32),
                  bias_offsets=i32(sums([len(b) for b in bias])))
    words = (vocab + 31) // 32
    table, place = None, [0] * rows
    if masks:
        table = np.random.default_rng(seed).integers(0, 2 ** 32, (3, words), dtype=np.uint64).astype(np.uint32)
        table[2] = 0
        place = [rng.randint(-1, 2) for _ in range(rows)]
        kw.update(mask=torch.from_numpy(table.view(np.int32)).cuda(), mask_rows=i32(place))
    assert dev.adjust_logits(x, out, tokens, stream=here(), **kw)
    torch.cuda.synchronize()
    import dev_reference as R

    for r in range(rows):
        allowed = None
        if masks and place[r] >= 0:
            bits = np.unpackbits(table[place[r]].view(np.uint8), bitorder="little")[:vocab].astype(bool)
            allowed = torch.from_numpy(bits)
        y, tol32, tol = R.logits(x0[r].cpu(), hist[r] if history else [], prompt[r], rep[r], pres[r], freq[r],
                                 bias[r] if biases else [], allowed, dt)
        R.check(out[r].cpu(), y, tol, f"row {r}")
        t = int(tokens[r])
        if not (y > -math.inf).any():
            assert t == -1, f"row {r}: nothing is allowed"
        else:
            best = y.nan_to_num(nan=-math.inf).max()
            assert 0 <= t < vocab and y[t] + 2 * tol32.max() >= best, f"row {r}: token {t}"


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 31), (3, 32), (5, 997), (2, 4096), (1, 70001), (4, 9973)])
def test_logits_match_64_bits(dev, dtype, rows, vocab):
    adjust_case(dev, dtype, rows, vocab, seed=rows * 1000 + vocab)


@pytest.mark.parametrize("history,biases,masks", [(0, 0, 0), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0)])
def test_logits_parts_alone(dev, history, biases, masks):
    adjust_case(dev, "f32", 3, 5000, 5, bool(history), bool(biases), bool(masks))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad", [1, 5, 8])
def test_logits_rows_off_16_bytes_in_place_and_padded(dev, dtype, pad):
    adjust_case(dev, dtype, 4, 3001, 9, in_place=True, pad=pad)
    adjust_case(dev, dtype, 4, 3001, 10, pad=pad)


def test_logits_long_history(dev):
    adjust_case(dev, "f32", 2, 151936, 11, hist_max=40000)


def test_logits_ties_infinities_and_nan(dev):
    torch = torch_()
    x = torch.zeros(6, 151936, device="cuda")
    x[0, [7, 70000, 151935]] = 5.0             # the lowest index of a tie
    x[1] = -math.inf                           # nothing above -inf
    x[2] = math.nan
    x[3] = math.nan
    x[3, 151935] = -3e38                       # NaN is above nothing
    x[4, 99] = math.inf
    x[4, 3] = math.nan
    x[5] = -1.0                                # a mask that allows NaN and infinity nowhere
    x[5, 10], x[5, 11] = math.nan, math.inf
    mask = torch.full((1, 4748), -1, dtype=torch.int32, device="cuda")
    mask[0, 0] = ~(3 << 10)
    out, tokens = torch.zeros_like(x), torch.zeros(6, dtype=torch.int32, device="cuda")
    assert dev.adjust_logits(x, out, tokens, mask=mask, mask_rows=i32([-1, -1, -1, -1, 1, 0]), stream=here())
    torch.cuda.synchronize()
    assert tokens.tolist() == [7, -1, -1, 151935, 99, 0]
    x[5, 10:12] = -math.inf
    assert torch.equal(out.nan_to_num(nan=4.0), x.nan_to_num(nan=4.0))


# --------------------------------------------------------- the rest of packed ----


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("sequences", [33, 300, 1500])
def test_packed_many_sequences(dev, dtype, sequences):
    """More sequences than a warp holds, many of them empty, some with fewer keys than queries."""
    torch = torch_()
    rng = random.Random(sequences)
    new = [rng.choice([0, 0, 1, 2, rng.randint(1, 40)]) for _ in range(sequences)]
    new[-1] = 5
    keys = [rng.choice([0, n, n + rng.randint(0, 90), max(0, n - 3)]) for n in new]
    dt = dtype_of(dtype)
    q, k, v = randn(1, sum(new), 4, 64, dtype=dt), randn(2, sum(keys), 2, 64, dtype=dt), randn(3, sum(keys), 2, 64, dtype=dt)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    qo, ko = i32(sums(new)), i32(sums(keys))
    assert dev.attention_packed(q, k, v, qo, ko, out, lse=lse, workspace=packed_space(dev, q, k, qo), stream=here())
    torch.cuda.synchronize()
    check_packed(q, k, v, new, keys, True, 0.125, out, lse)
    dev.status()


@pytest.mark.parametrize("dtype,heads,kv_heads,size,new,keys,causal", [
    ("f16", 8, 1, 128, [1], [9000], True),
    ("bf16", 4, 4, 64, [3, 1], [5000, 4100], True),
    ("f16", 6, 2, 96, [40], [40 + 6000], True),
    ("bf16", 2, 1, 128, [260], [3000], False),
    ("f16", 2, 1, 40, [100, 1], [2100, 6000], True),
    ("f16", 12, 4, 112, [2, 0, 37], [901, 333, 1020], True),  # short ones, with one tile of rows a CTA
    ("bf16", 16, 16, 32, [1, 2], [1023, 777], False),
    ("bf16", 8, 8, 128, [130], [1000], True),
])
def test_packed_keys_cut_into_parts(dev, dtype, heads, kv_heads, size, new, keys, causal):
    """Few rows and many keys: the call is cut over the keys and joined; rows of no sequence stay as they were."""
    torch = torch_()
    dt = dtype_of(dtype)
    total = sum(new) + 3
    q = randn(1, total, heads, size, dtype=dt)
    k, v = randn(2, sum(keys), kv_heads, size, dtype=dt), randn(3, sum(keys), kv_heads, size, dtype=dt)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    qo, ko = i32([2 + n for n in sums(new)]), i32(sums(keys))
    assert dev.attention_packed_workspace(q, k, qo) > 0
    assert dev.attention_packed(q, k, v, qo, ko, out, causal=causal, lse=lse, workspace=packed_space(dev, q, k, qo),
                                stream=here())
    torch.cuda.synchronize()
    check_packed(q, k, v, new, keys, causal, size ** -0.5, out, lse, start=(2, 0))
    for t in (out, lse):
        assert (t[:2] == 7.0).all() and (t[total - 1:] == 7.0).all()
    dev.status()


@pytest.mark.parametrize("size,keys", [(128, 300), (64, 300), (128, 6000), (128, 900)])
def test_packed_masked_keys_that_are_not_finite(dev, size, keys):
    """Keys and values behind the causal border are infinite or NaN: the queries before them do not see them, and those
    at and after them do."""
    torch = torch_()
    new, at = 40, keys - 17
    q, k, v = randn(1, new, 4, size, dtype=torch.float16), *(randn(i, keys, 2, size, dtype=torch.float16) for i in (2, 3))
    k[at], v[at, 0], v[at + 3, 1, 5] = math.nan, math.inf, math.nan
    out, lse = torch.zeros_like(q), torch.zeros(new, 4, device="cuda")
    qo, ko = i32([0, new]), i32([0, keys])
    assert dev.attention_packed(q, k, v, qo, ko, out, lse=lse, workspace=packed_space(dev, q, k, qo), stream=here())
    torch.cuda.synchronize()
    seen = new - 17  # the first query that sees key `at`
    import dev_reference as R

    want = R.attention(q[:seen], k[:at], v[:at], size ** -0.5, visible(new, keys, True)[:seen, :at], q.dtype)
    R.check(out[:seen], want[0], want[2], "out")
    R.check(lse[:seen], want[1], want[3], "lse")
    assert torch.isnan(out[seen:]).all() and torch.isnan(lse[seen:]).all()
    # Values alone: only the channels that they reach.
    k[at] = 0.5
    v[at, 0] = 1.0
    assert dev.attention_packed(q, k, v, qo, ko, out, lse=lse, workspace=packed_space(dev, q, k, qo), stream=here())
    torch.cuda.synchronize()
    bad = torch.isnan(out)
    assert bad[seen + 3:, 2:, 5].all()
    bad[seen + 3:, 2:, 5] = False
    assert not bad.any()
    check_packed(q[:seen + 3], k[:at + 3], v[:at + 3], [seen + 3], [at + 3], True, size ** -0.5, out[:seen + 3], lse[:seen + 3])


def test_packed_broadcast_heads_and_offsets_beyond_32_bits(dev):
    """K and V expanded over heads (stride 0) are read in place or declined; a cache whose token stride passes 2^31
    elements over its length is read where it lies."""
    torch = torch_()
    q = randn(1, 50, 4, 64, dtype=torch.float16)
    k1, v1 = randn(2, 70, 1, 64, dtype=torch.float16), randn(3, 70, 1, 64, dtype=torch.float16)
    k, v = k1.expand(70, 4, 64), v1.expand(70, 4, 64)
    out, lse = torch.full_like(q, 7.0), torch.zeros(50, 4, device="cuda")
    qo, ko = i32([0, 50]), i32([0, 70])
    if dev.attention_packed(q, k, v, qo, ko, out, lse=lse, workspace=packed_space(dev, q, k, qo), stream=here()):
        torch.cuda.synchronize()
        check_packed(q, k, v, [50], [70], True, 0.125, out, lse)
    else:
        assert (out == 7.0).all()
    store = torch.zeros(70 * (1 << 26), dtype=torch.float16, device="cuda")
    far = store.as_strided((70, 1, 64), (1 << 26, 64, 1))
    far.copy_(k1)
    assert dev.attention_packed(q, far, v1, qo, ko, out, lse=lse, workspace=packed_space(dev, q, far, qo), stream=here())
    torch.cuda.synchronize()
    check_packed(q, far, v1, [50], [70], True, 0.125, out, lse)


def test_shared_offsets_beyond_32_bits(dev):
    torch = torch_()
    store = torch.zeros(2 * (1 << 31) + 4096, dtype=torch.float16, device="cuda")
    sk = store.as_strided((3, 30, 1, 64), ((1 << 31), 64, 64, 1))
    sk.copy_(randn(1, 3, 30, 1, 64, dtype=torch.float16))
    sv, q = randn(2, 3, 30, 1, 64, dtype=torch.float16), randn(3, 3, 2, 64, dtype=torch.float16)
    pk, pv = randn(4, 10, 1, 64, dtype=torch.float16), randn(5, 10, 1, 64, dtype=torch.float16)
    out, lse = torch.zeros_like(q), torch.zeros(3, 2, device="cuda")
    assert dev.attention_shared(q, pk, pv, sk, sv, i32([30, 7, 22]), out, lse=lse, workspace=shared_space(dev, q, pk, sk),
                                stream=here())
    torch.cuda.synchronize()
    check_shared(q, pk, pv, sk, sv, [30, 7, 22], 0.125, out, lse)


def test_wrong_offsets_and_lengths_stay_in_bounds(dev):
    """Offsets that decrease or pass the arrays, and lengths beyond the capacity, are clamped; the guard rows hold."""
    torch = torch_()
    q, k, v = (randn(i, 60, 2, 64, dtype=torch.float16) for i in range(3))
    out = torch.full((64, 2, 64), 7.0, dtype=torch.float16, device="cuda")
    for qo, ko in (([0, 50, 20, 90], [0, 80, -5, 60]), ([-3, 10, 10, 60], [0, 10, 70, 65]), ([60, 0, 60, 60], [60, 0, 0, 60])):
        assert dev.attention_packed(q, k, v, i32(qo), i32(ko), out[2:62], stream=here(),
                                    workspace=packed_space(dev, q, k, i32(qo)))
    torch.cuda.synchronize()
    assert (out[:2] == 7.0).all() and (out[62:] == 7.0).all()
    sk = randn(4, 60, 9, 2, 64, dtype=torch.float16)
    lens = i32([40, -3] * 30)
    lse = torch.zeros(60, 2, device="cuda")
    assert dev.attention_shared(q, k, v, sk, sk, lens, out[2:62], lse=lse, workspace=shared_space(dev, q, k, sk), stream=here())
    torch.cuda.synchronize()
    check_shared(q, k, v, sk, sk, [9, 0] * 30, 0.125, out[2:62], lse)
    x = randn(5, 4, 100, dtype=torch.float32)
    y = torch.full((6, 100), 7.0, device="cuda")
    assert dev.adjust_logits(x, y[1:5], None, history=i32([5, 6, 7]), history_offsets=i32([-2, 3, 1, 9, 2]),
                             bias_tokens=i32([1]), bias_values=torch.ones(1, device="cuda"), bias_offsets=i32([0, 5, -1, 1, 1]),
                             stream=here())
    torch.cuda.synchronize()
    assert (y[0] == 7.0).all() and (y[5] == 7.0).all()
    dev.status()


# ----------------------------------------------------------- streams and graphs ----


def test_streams_none_two_at_once_and_threads(dev):
    """The backend's own stream; two streams with a workspace each; two host threads."""
    import threading

    torch = torch_()
    q, k, v = randn(1, 30, 8, 128, dtype=torch.bfloat16), *(randn(i, 9000, 1, 128, dtype=torch.bfloat16) for i in (2, 3))
    qo, ko = i32([0, 30]), i32([0, 9000])
    outs = [torch.zeros_like(q) for _ in range(5)]
    spaces = [packed_space(dev, q, k, qo) for _ in range(5)]
    torch.cuda.synchronize()
    assert dev.attention_packed(q, k, v, qo, ko, outs[0], workspace=spaces[0])  # the backend's own stream
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i, s in enumerate(streams):
        assert dev.attention_packed(q, k, v, qo, ko, outs[1 + i], workspace=spaces[1 + i], stream=s.cuda_stream)

    def work(i):
        for _ in range(20):
            assert dev.attention_packed(q, k, v, qo, ko, outs[3 + i], workspace=spaces[3 + i], stream=streams[i].cuda_stream)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    dev.status()  # waits for the device
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


def test_a_decode_step_of_the_three_operators_captured_and_replayed(dev):
    """Two prompts prefilled in one packed call, then decode steps of both on the shared prefix with their logits
    adjusted, captured once and replayed with other lengths, tokens and histories in the same buffers."""
    import dev_reference as R

    torch = torch_()
    heads, kv_heads, size, prefix, cap, vocab, n = 4, 2, 64, 300, 50, 2000, 6
    dt = torch.bfloat16
    # Prefill: the shared prompt and one more prompt, packed.
    pq, pk, pv = randn(1, prefix + 40, heads, size, dtype=dt), *(randn(i, prefix + 40, kv_heads, size, dtype=dt) for i in (2, 3))
    off = i32([0, prefix, prefix + 40])
    pout, plse = torch.zeros_like(pq), torch.zeros(prefix + 40, heads, device="cuda")
    assert dev.attention_packed(pq, pk, pv, off, off, pout, lse=plse, workspace=packed_space(dev, pq, pk, off), stream=here())
    torch.cuda.synchronize()
    check_packed(pq, pk, pv, [prefix, 40], [prefix, 40], True, 0.125, pout, plse)

    # Decode: n sessions on the first prompt's keys.
    k0, v0 = pk[:prefix], pv[:prefix]
    sk, sv = (randn(i, n, cap, kv_heads, size, dtype=dt) for i in (4, 5))
    q, lens = torch.zeros(n, heads, size, dtype=dt, device="cuda"), i32([0] * n)
    out, lse = torch.zeros_like(q), torch.zeros(n, heads, device="cuda")
    head = randn(6, heads * size, vocab, dtype=dt)
    logits, adjusted, tokens = (torch.zeros(n, vocab, dtype=dt, device="cuda"), torch.zeros(n, vocab, dtype=dt, device="cuda"),
                                i32([0] * n))
    history, hoff = i32([0] * 60), i32([0] * (n + 1))
    rep, pres, freq = (torch.full((n,), x, device="cuda") for x in (1.3, 0.2, 0.1))
    space = shared_space(dev, q, k0, sk)

    def step():
        stream = here()
        assert dev.attention_shared(q, k0, v0, sk, sv, lens, out, lse=lse, workspace=space, stream=stream)
        torch.mm(out.view(n, -1), head, out=logits)
        assert dev.adjust_logits(logits, adjusted, tokens, history=history, history_offsets=hoff, repetition=rep,
                                 presence=pres, frequency=freq, stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    rng = random.Random(3)
    for turn in range(3):
        own = [rng.randint(0, cap) for _ in range(n)]
        hist = [[rng.randrange(vocab) for _ in range(rng.randint(0, 10))] for _ in range(n)]
        q.copy_(randn(10 + turn, n, heads, size, dtype=dt))
        lens.copy_(i32(own))
        flat = [t for h in hist for t in h]
        history[:len(flat)].copy_(i32(flat) if flat else history[:0])
        hoff.copy_(i32(sums([len(h) for h in hist])))
        graph.replay()
        torch.cuda.synchronize()
        check_shared(q, k0, v0, sk, sv, own, 0.125, out, lse)
        for r in range(n):
            y, tol32, tol = R.logits(logits[r].cpu(), hist[r], 0, np.float32(1.3).item(), np.float32(0.2).item(),
                                     np.float32(0.1).item(), [], None, dt)
            R.check(adjusted[r].cpu(), y, tol, f"turn {turn} row {r}")
            assert y[int(tokens[r])] + 2 * tol32.max() >= y.max()
    dev.status()


def test_results_do_not_change_from_call_to_call(dev):
    torch = torch_()
    q, k, v = randn(1, 300, 16, 128, dtype=torch.float16), *(randn(i, 5000, 2, 128, dtype=torch.float16) for i in (2, 3))
    qo, ko = i32([0, 100, 300]), i32([0, 2000, 5000])
    outs = []
    for _ in range(4):
        out, lse = torch.zeros_like(q), torch.zeros(300, 16, device="cuda")
        assert dev.attention_packed(q, k, v, qo, ko, out, lse=lse, workspace=packed_space(dev, q, k, qo), stream=here())
        sout, slse = torch.zeros(20, 16, 128, dtype=q.dtype, device="cuda"), torch.zeros(20, 16, device="cuda")
        sk = k[:4000].view(20, 200, 2, 128)
        assert dev.attention_shared(q[:20], k, v, sk, sk, i32(list(range(20))), sout, lse=slse,
                                    workspace=shared_space(dev, q[:20], k, sk), stream=here())
        x = q[:40].float().reshape(40, -1)
        y, t = torch.zeros_like(x), i32([0] * 40)
        assert dev.adjust_logits(x, y, t, history=i32([3, 3, 9] * 40), history_offsets=i32([3 * i for i in range(41)]),
                                 frequency=torch.ones(40, device="cuda"), stream=here())
        torch.cuda.synchronize()
        outs.append((out, lse, sout, slse, y, t))
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


@pytest.mark.parametrize("rows,vocab", [(160, 5000), (160, 70001), (40, 33000)])
def test_logits_more_rows_than_the_gpu_has_sms(dev, rows, vocab):
    adjust_case(dev, "bf16", rows, vocab, 21, hist_max=30)


def test_logits_more_tokens_than_slots(dev):
    """A history and biases that touch more tokens than a CTA's table holds, in one row of several."""
    adjust_case(dev, "f32", 3, 9000, 22, hist_max=30000)
    torch = torch_()
    x = randn(1, 200, 9000, dtype=torch.float32)
    every = torch.arange(9000, dtype=torch.int32, device="cuda")
    y, t = torch.zeros_like(x), i32([0] * 200)
    # Row 7 biases every token twice (the later entry counts) and lists every token in its history.
    off = i32([0] * 8 + [9000] * 193)
    assert dev.adjust_logits(x, y, t, history=every, history_offsets=off, presence=torch.full((200,), 0.5, device="cuda"),
                             bias_tokens=torch.cat([every, every]), bias_offsets=i32([0] * 8 + [18000] * 193),
                             bias_values=torch.cat([torch.full((9000,), 99.0, device="cuda"), every.float() / 64]), stream=here())
    torch.cuda.synchronize()
    want = x.clone()
    want[7] = (x[7] - 0.5) + every.float() / 64
    assert torch.equal(y, want) and torch.equal(t.long(), want.argmax(-1))
