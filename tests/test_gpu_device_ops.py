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
