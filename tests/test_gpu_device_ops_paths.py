"""Paths of the device-pointer operators that depend on a call's sizes, each pinned to the path that it is for."""
import math
import random

import pytest
from test_gpu_device_ops import (adjust_case, check_packed, check_shared, dev, dtype_of, here, i32, packed_space,  # noqa: F401
                                 randn, shared_space, sums, torch_)

pytestmark = pytest.mark.gpu


# ------------------------------------------- packed: two row tiles a CTA, keys not cut ----


def packed_uncut(dev, q, k, v, new, keys, causal=True, scale=None):
    """One call that takes two row tiles a CTA (more than 1024 keys a sequence on average) and cuts no keys."""
    torch = torch_()
    assert sum(keys) > 1024 * len(keys)
    qo, ko = i32(sums(new)), i32(sums(keys))
    assert dev.attention_packed_workspace(q, k, qo) == 0
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    assert dev.attention_packed(q, k, v, qo, ko, out, causal=causal, scale=scale, lse=lse, stream=here())
    torch.cuda.synchronize()
    dev.status()
    return out, lse


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,size,new,keys,causal", [
    (16, 8, 128, [1500, 2300], None, True),
    (14, 2, 64, [1500, 2300], None, True),          # seven heads a group: rows of a tile that carry no query
    (24, 8, 96, [1900, 2100], None, True),          # three
    (20, 20, 80, [1300, 1700], [1250, 1700], True),  # the first 50 queries see no key
    (32, 32, 40, [1300, 1701], [1250, 1999], False),
    (16, 16, 64, [1600], None, True),
    (64, 1, 112, [1200], [1300], True),
])
def test_packed_two_tiles_uncut_matches_64_bits(dev, dtype, heads, kv_heads, size, new, keys, causal):
    keys = new if keys is None else keys
    dt = dtype_of(dtype)
    q, k, v = (randn(1 + i, sum(n), h, size, dtype=dt) for i, (n, h) in enumerate(((new, heads), (keys, kv_heads), (keys, kv_heads))))
    out, lse = packed_uncut(dev, q, k, v, new, keys, causal)
    check_packed(q, k, v, new, keys, causal, size ** -0.5, out, lse)


@pytest.mark.parametrize("heads,kv_heads,size", [(8, 8, 32), (8, 4, 128)])
def test_packed_two_tiles_uncut_many_sequences(dev, heads, kv_heads, size):
    """More sequences than a warp holds, empty ones among them, with fewer and with more keys than queries."""
    rng = random.Random(2)
    new = [rng.choice([0, 1, rng.randint(1, 300), 130]) for _ in range(40)]
    keys = [rng.choice([0, n + rng.randint(1200, 2500), 1800, max(0, n - 3)]) for n in new]
    new[7], keys[7], keys[8] = 290, 280, 6000
    q, k, v = (randn(1 + i, sum(n), h, size, dtype=dtype_of("bf16"))
               for i, (n, h) in enumerate(((new, heads), (keys, kv_heads), (keys, kv_heads))))
    out, lse = packed_uncut(dev, q, k, v, new, keys)
    check_packed(q, k, v, new, keys, True, size ** -0.5, out, lse)


@pytest.mark.parametrize("size", [64, 128])
def test_packed_two_tiles_uncut_scores_that_rise(dev, size):
    """Scores that rise by hundreds along the keys: the running maximum moves at every step and O is rescaled."""
    torch = torch_()
    n, dt = 1600, dtype_of("bf16")
    q, v = randn(7, n, 16, size, dtype=dt), randn(9, n, 16, size, dtype=dt)
    k = randn(8, n, 16, size, dtype=dt) * torch.linspace(0.1, 20, n, device="cuda")[:, None, None].bfloat16()
    out, lse = packed_uncut(dev, q, k, v, [n], [n], scale=1.0)
    check_packed(q, k, v, [n], [n], True, 1.0, out, lse)


@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("at", [1189, 1252, 1283])
def test_packed_two_tiles_uncut_masked_keys_that_are_not_finite(dev, size, at):
    """Key `at` and values from it on are not finite: rows before it, in the tile that ends just before it, in the one
    that takes it in behind its border and in other CTAs, do not see them."""
    torch = torch_()
    new, keys = 1200, 1300
    q, k, v = randn(1, new, 16, size, dtype=dtype_of("f16")), *(randn(i, keys, 16, size, dtype=dtype_of("f16")) for i in (2, 3))
    seen = at - (keys - new)  # the first query that sees key `at`
    k[at, :8], v[at, :8], v[at + 5, 8:, 5] = math.nan, math.inf, math.nan
    out, lse = packed_uncut(dev, q, k, v, [new], [keys])
    check_packed(q[:seen], k[:at], v[:at], [seen], [at], True, size ** -0.5, out[:seen], lse[:seen])
    assert torch.isnan(out[seen:, :8]).all() and torch.isnan(lse[seen:, :8]).all()
    bad = torch.isnan(out[:, 8:])
    assert bad[seen + 5:, :, 5].all()
    bad[seen + 5:, :, 5] = False
    assert not bad.any()
    check_packed(q[:seen + 5, 8:], k[:at + 5, 8:], v[:at + 5, 8:], [seen + 5], [at + 5], True, size ** -0.5, out[:seen + 5, 8:],
                 lse[:seen + 5, 8:])


# ------------------------------------------------ shared: caches with room for more ----


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,size,prefix,lens,cap,joined", [
    (16, 8, 128, 61, [0, 7], 4096, True),                     # sixteen ranges of a row, almost all of them empty
    (16, 8, 128, 0, [0, 0, 5], 8192, True),
    (32, 8, 128, 6, [0, 1, 3, 70, 0], 800, False),            # ranges joined in a cluster, some without a stage
    (8, 1, 112, 0, [0, 65, 0, 1], 900, False),
    (14, 2, 64, 40, [0, 2], 1500, False),
    (16, 8, 128, 2048, [0, 664, 1] + [10 * i for i in range(61)], 4096, True),  # the prefix on the tensor cores
    (32, 4, 64, 5000, [0, 1, 70, 33] * 20, 1000, True),
])
def test_shared_capacity_far_above_the_lengths(dev, dtype, heads, kv_heads, size, prefix, lens, cap, joined):
    torch = torch_()
    n, dt = len(lens), dtype_of(dtype)
    q, out = randn(1, n, heads, size, dtype=dt), torch.full((n, heads, size), 7.0, dtype=dt, device="cuda")
    pk, pv = randn(2, prefix, kv_heads, size, dtype=dt), randn(3, prefix, kv_heads, size, dtype=dt)
    sk, sv = (torch.full((n, cap, kv_heads, size), math.nan, dtype=dt, device="cuda") for _ in range(2))
    for b, m in enumerate(lens):
        sk[b, :m], sv[b, :m] = randn(4 + 2 * b, m, kv_heads, size, dtype=dt), randn(5 + 2 * b, m, kv_heads, size, dtype=dt)
    lse = torch.full((n, heads), 7.0, device="cuda")
    assert (dev.attention_shared_workspace(q, pk, sk) > 0) == joined
    assert dev.attention_shared(q, pk, pv, sk, sv, i32(lens), out, lse=lse, workspace=shared_space(dev, q, pk, sk),
                                stream=here())
    torch.cuda.synchronize()
    check_shared(q, pk, pv, sk, sv, lens, size ** -0.5, out, lse)
    dev.status()


# -------------------------------------------------- logits: large vocabularies, ties ----


@pytest.mark.parametrize("dtype,rows,vocab,history", [
    ("bf16", 80, (1 << 20) + 1, 40),       # rows enough for the GPU, cut all the same
    ("f16", 75, 1 << 20, 16000),           # the longest part of a CTA, its table overflows in some rows
    ("f32", 1, 1 << 24, 4000),             # a cluster of the largest parts
    ("bf16", 2, (1 << 24) - 5, 60000),     # whose tables overflow
    ("f32", 30, (1 << 21) + 33, 300),
])
def test_logits_large_vocabularies(dev, monkeypatch, dtype, rows, vocab, history):
    import dev_reference as R

    def check(got, want, tol, what):
        """R.check without its quotient: among so many logits one is exactly 0, its bound is 0, and 0 / 0 is NaN."""
        got, want = got.double(), want.double()
        assert torch_().equal(torch_().isnan(got), torch_().isnan(want)), f"{what}: NaN in other places"
        fine = torch_().isfinite(want)
        assert torch_().equal(got[~fine & ~torch_().isnan(want)], want[~fine & ~torch_().isnan(want)]), f"{what}: infinities differ"
        assert ((got - want).abs()[fine] <= tol.expand_as(want)[fine]).all(), f"{what}: outside the bound"

    monkeypatch.setattr(R, "check", check)
    adjust_case(dev, dtype, rows, vocab, 31, hist_max=history)


@pytest.mark.parametrize("rows,vocab", [(1, 151936), (40, 151936), (100, 151936), (3, 4097)])
def test_logits_ties_between_touched_and_untouched_tokens(dev, rows, vocab):
    """Equal values of a token of the history, one of the biases and one of neither, in one CTA's part and in several:
    the lowest index wins.  All values are exact."""
    torch = torch_()
    last = vocab - 1
    places = [(3, 5, 7), (5, 3, 7), (7, 5, 3), (3, last, 9), (last, 3, 9), (9, last, 3), (vocab // 2, vocab // 2 - 1, last),
              (vocab // 2 - 1, vocab // 2, last), (last, last - 1, last - 2), (0, last, vocab // 3), (last, 0, vocab // 3),
              (vocab // 3, last, 0), (4096, 2048, 1024)]
    for start in range(len(places)):
        mine = [places[(start + r) % len(places)] for r in range(rows)]
        x = torch.full((rows, vocab), -1.0, device="cuda")
        for r, (touched, biased, free) in enumerate(mine):
            x[r, touched], x[r, free] = 4.0, 2.0
        out, tokens = torch.zeros_like(x), i32([0] * rows)
        assert dev.adjust_logits(x, out, tokens, history=i32([p[0] for p in mine]), history_offsets=i32(list(range(rows + 1))),
                                 repetition=torch.full((rows,), 2.0, device="cuda"), bias_tokens=i32([p[1] for p in mine]),
                                 bias_values=torch.full((rows,), 3.0, device="cuda"),
                                 bias_offsets=i32(list(range(rows + 1))), stream=here())
        torch.cuda.synchronize()
        assert tokens.tolist() == [min(p) for p in mine]
        for r, p in enumerate(mine):
            assert (out[r, list(p)] == 2.0).all()


# ------------------------------------------------------ one workspace for all batches ----


def test_one_workspace_serves_a_batch_that_shrinks(dev):
    """Sessions end and prompts arrive in other numbers: a workspace of the bound's size, and not a byte more, is enough."""
    torch = torch_()
    heads, kv_heads, size, dt = 16, 8, 128, dtype_of("bf16")

    def guarded(n):
        store = torch.full((n + 256,), 77, dtype=torch.uint8, device="cuda")
        return store[:n], store[n:]

    prefix, cap, most = 2048, 4000, 6
    space, guard = guarded(dev.attention_shared_workspace_bound(prefix, cap, most, heads, kv_heads, size))
    q, pk, pv = randn(1, most, heads, size, dtype=dt), *(randn(i, prefix, kv_heads, size, dtype=dt) for i in (2, 3))
    sk, sv = (randn(i, most, cap, kv_heads, size, dtype=dt) for i in (4, 5))
    lens = [70, 4000, 0, 999, 1, 333]
    for n in range(most, 0, -1):
        out, lse = torch.zeros_like(q[:n]), torch.zeros(n, heads, device="cuda")
        assert dev.attention_shared(q[:n], pk, pv, sk[:n], sv[:n], i32(lens[:n]), out, lse=lse, workspace=space, stream=here())
        torch.cuda.synchronize()
        check_shared(q[:n], pk, pv, sk[:n], sv[:n], lens[:n], size ** -0.5, out, lse)
        assert (guard == 77).all()
    total_q, total_k = 400, 9000
    space, guard = guarded(dev.attention_packed_workspace_bound(total_q, total_k, heads, kv_heads, size))
    q, k, v = randn(1, total_q, heads, size, dtype=dt), *(randn(i, total_k, kv_heads, size, dtype=dt) for i in (2, 3))
    for new, keys in (([400], [9000]), ([300], [1000]), ([100], [1000]), ([1], [9000]), ([64, 1, 7], [64, 6000, 77])):
        a, b = sum(new), sum(keys)
        out, lse = torch.zeros_like(q[:a]), torch.zeros(a, heads, device="cuda")
        assert dev.attention_packed(q[:a], k[:b], v[:b], i32(sums(new)), i32(sums(keys)), out, lse=lse, workspace=space,
                                    stream=here())
        torch.cuda.synchronize()
        check_packed(q[:a], k[:b], v[:b], new, keys, True, size ** -0.5, out, lse)
        assert (guard == 77).all()
