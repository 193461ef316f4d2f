"""Refusals of the device-pointer operators: arguments are checked before the backend, so no device is needed.

The structs are filled from Python as a host in another language fills them, which also pins their layout."""
import ctypes as C
import math

import pytest

OK, DECLINED, ARGUMENT = 0, 1, -1
F32, F16, BF16 = 0, 1, 2
P, I64, I32, F = C.c_void_p, C.c_int64, C.c_int32, C.c_float


class Packed(C.Structure):
    _fields_ = [("q", P), ("k", P), ("v", P), ("out", P), ("lse", P), ("q_offsets", P), ("k_offsets", P), ("workspace", P),
                ("workspace_bytes", I64), ("q_stride", I64 * 2), ("k_stride", I64 * 2), ("v_stride", I64 * 2),
                ("out_stride", I64 * 2), ("total_q", I64), ("total_k", I64), ("dtype", I32), ("sequences", I32),
                ("heads", I32), ("kv_heads", I32), ("head_size", I32), ("causal", I32), ("scale", F), ("reserved", I32)]


class Shared(C.Structure):
    _fields_ = [("q", P), ("prefix_k", P), ("prefix_v", P), ("suffix_k", P), ("suffix_v", P), ("out", P), ("lse", P),
                ("suffix_lens", P), ("workspace", P), ("workspace_bytes", I64), ("q_stride", I64 * 2),
                ("prefix_k_stride", I64 * 2), ("prefix_v_stride", I64 * 2), ("suffix_k_stride", I64 * 3),
                ("suffix_v_stride", I64 * 3), ("out_stride", I64 * 2), ("prefix_len", I64), ("suffix_capacity", I64),
                ("dtype", I32), ("sequences", I32), ("heads", I32), ("kv_heads", I32), ("head_size", I32), ("scale", F)]


class Logits(C.Structure):
    _fields_ = [(n, P) for n in ("logits", "out", "tokens", "history", "history_offsets", "prompt_lens", "repetition",
                                 "presence", "frequency", "bias_tokens", "bias_values", "bias_offsets", "mask", "mask_rows")]
    _fields_ += [("logits_stride", I64), ("out_stride", I64), ("mask_stride", I64), ("history_total", I64),
                 ("bias_total", I64), ("dtype", I32), ("rows", I32), ("vocab", I32), ("mask_count", I32)]


def packed(**kw):
    a = Packed(q=1 << 20, k=1 << 21, v=1 << 22, out=1 << 23, q_offsets=64, k_offsets=64, workspace=1 << 24,
               workspace_bytes=1 << 40, q_stride=(2048, 128), k_stride=(1024, 128), v_stride=(1024, 128),
               out_stride=(2048, 128), total_q=100, total_k=100, dtype=F16, sequences=3, heads=16, kv_heads=8, head_size=128,
               causal=1, scale=0.1)
    return fill(a, kw)


def shared(**kw):
    a = Shared(q=1 << 20, prefix_k=1 << 21, prefix_v=1 << 22, suffix_k=1 << 21, suffix_v=1 << 22, out=1 << 23, suffix_lens=64,
               workspace=1 << 24, workspace_bytes=1 << 40, q_stride=(2048, 128), prefix_k_stride=(1024, 128),
               prefix_v_stride=(1024, 128), suffix_k_stride=(102400, 1024, 128), suffix_v_stride=(102400, 1024, 128),
               out_stride=(2048, 128), prefix_len=500, suffix_capacity=100, dtype=BF16, sequences=3, heads=16, kv_heads=8,
               head_size=128, scale=0.1)
    return fill(a, kw)


def logits(**kw):
    a = Logits(logits=1 << 20, out=1 << 22, tokens=64, logits_stride=1000, out_stride=1000, dtype=F32, rows=4, vocab=1000)
    return fill(a, kw)


def fill(a, kw):
    for name, value in kw.items():
        field = getattr(a, name)
        setattr(a, name, type(field)(*value) if isinstance(value, tuple) else value)
    return a


@pytest.fixture(scope="module")
def call(built_lib):
    from funasrnet_b200._lib import lib

    def go(args):
        fn = {Packed: "fa_dev_attention_packed", Shared: "fa_dev_attention_shared", Logits: "fa_dev_adjust_logits"}[type(args)]
        rc = getattr(lib(), fn)(None, C.byref(args), None)
        return rc, lib().fa_last_error().decode() if rc < 0 else ""

    return go


def test_struct_sizes():
    assert (C.sizeof(Packed), C.sizeof(Shared), C.sizeof(Logits)) == (184, 232, 168)


@pytest.mark.parametrize("make", [packed, shared, logits])
def test_well_formed_arguments_reach_the_backend(call, make):
    assert call(make()) == (ARGUMENT, "null backend")


BAD = [
    (packed, dict(dtype=7), "dtype"),
    (packed, dict(heads=15), "multiple of kv_heads"),
    (packed, dict(kv_heads=0), "positive"),
    (packed, dict(sequences=-1), "sequence"),
    (packed, dict(total_q=-1), "negative"),
    (packed, dict(scale=0.0), "scale"),
    (packed, dict(scale=math.nan), "scale"),
    (packed, dict(scale=-1.0), "scale"),
    (packed, dict(q=None), "null"),
    (packed, dict(k_offsets=None), "null"),
    (packed, dict(v=None), "null"),
    (packed, dict(q_stride=(-2048, 128)), "stride"),
    (packed, dict(out_stride=(128, 128)), "overlap"),
    (packed, dict(out_stride=(2048, 0)), "overlap"),
    (packed, dict(reserved=1), "reserved"),
    (packed, dict(total_q=1, total_k=9000, sequences=1, workspace_bytes=16), "workspace"),
    (packed, dict(total_q=1, total_k=9000, sequences=1, workspace=8), "workspace"),
    (shared, dict(prefix_len=-1), "negative"),
    (shared, dict(prefix_v=None), "null"),
    (shared, dict(suffix_lens=None), "null"),
    (shared, dict(out=None), "null"),
    (shared, dict(out_stride=(64, 128)), "overlap"),
    (shared, dict(sequences=64, prefix_len=9000, workspace_bytes=0), "workspace"),
    (packed, dict(out_stride=(1 << 37, (1 << 38) - 8), total_q=(1 << 27) - 1), "overlap"),
    (logits, dict(rows=1 << 27, logits_stride=1 << 38, out_stride=1 << 38), "stride"),
    (logits, dict(rows=-1), "rows"),
    (logits, dict(vocab=0), "vocab"),
    (logits, dict(logits=None), "null"),
    (logits, dict(logits_stride=999), "overlap"),
    (logits, dict(out_stride=10), "overlap"),
    (logits, dict(history=64), "history_offsets"),
    (logits, dict(bias_tokens=64, bias_values=64), "bias"),
    (logits, dict(history_total=1 << 31), "history_total"),
    (logits, dict(mask=64, mask_stride=32, mask_count=3), "fewer mask rows"),
    (logits, dict(mask=64, mask_stride=3, mask_count=9), "mask rows overlap"),
    (logits, dict(out=(1 << 20) + 4), "overlaps"),
    (logits, dict(out=1 << 20, out_stride=2000), "overlaps"),
]


@pytest.mark.parametrize("make,change,word", BAD)
def test_inconsistent_arguments_are_refused(call, make, change, word):
    rc, message = call(make(**change))
    assert rc == ARGUMENT and word in message, message


@pytest.mark.parametrize("make,change", [
    (packed, dict(dtype=F32)),
    (packed, dict(head_size=136)),
    (packed, dict(head_size=100)),
    (packed, dict(heads=130, kv_heads=1)),
    (packed, dict(total_k=1 << 30)),
    (packed, dict(total_q=1 << 28)),
    (packed, dict(total_q=1 << 62)),
    (packed, dict(sequences=1 << 28)),  # more CTAs than a grid has
    (packed, dict(q=(1 << 20) + 8)),
    (packed, dict(k_stride=(1028, 128))),
    (shared, dict(dtype=F32)),
    (shared, dict(head_size=12)),
    (shared, dict(suffix_v=(1 << 22) + 2)),
    (shared, dict(suffix_k_stride=(102401, 1024, 128))),
    (shared, dict(suffix_capacity=1 << 30)),
    (shared, dict(prefix_len=(1 << 63) - 1)),
    (logits, dict(vocab=(1 << 24) + 1, logits_stride=1 << 25, out_stride=1 << 25)),
])
def test_sizes_outside_the_kernels_are_declined(call, make, change):
    assert call(make(**change))[0] == DECLINED


@pytest.mark.parametrize("make,change", [
    (packed, dict(total_q=1, q_stride=(5, 128), out_stride=(3, 128))),
    (packed, dict(heads=1, kv_heads=1, q_stride=(128, 1), k_stride=(128, 3), out_stride=(128, 1))),
    (shared, dict(sequences=1, suffix_k_stride=(7, 1024, 128))),
    (logits, dict(out=(1 << 20) + 4000, logits_stride=2000, out_stride=2000)),  # side by side in one array
    (logits, dict(out=1 << 20)),                                                # in place
    (logits, dict(rows=1, logits_stride=1, out_stride=0)),
])
def test_strides_without_a_say_and_outputs_beside_the_input(call, make, change):
    assert call(make(**change)) == (ARGUMENT, "null backend")  # nothing else is wrong


def test_null_arguments_and_empty_calls(built_lib, call):
    from funasrnet_b200._lib import lib

    assert lib().fa_dev_attention_packed(None, None, None) == ARGUMENT
    assert lib().fa_dev_adjust_logits(None, None, None) == ARGUMENT
    assert lib().fa_dev_status(None) == ARGUMENT
    for args in (packed(total_q=0, q=None, out=None), packed(sequences=0, q_offsets=None), shared(sequences=0, q=None, out=None),
                 logits(rows=0, logits=None)):
        assert call(args) == (ARGUMENT, "null backend")  # nothing else is wrong


def test_workspace_sizes(built_lib):
    from funasrnet_b200._lib import lib

    size = lib().fa_dev_attention_packed_workspace
    assert size(8192, 8192, 1, 16, 8, 128) == 0
    assert size(1, 20000, 1, 16, 8, 128) >= 2 * 16 * 128 * 4
    assert size(0, 0, 0, 16, 8, 128) == 0 and size(5, 5, 1, 15, 8, 128) == 0 and size(-1, 5, 1, 8, 8, 128) == 0
    size = lib().fa_dev_attention_shared_workspace
    assert size(0, 10, 2, 16, 8, 128) == 0
    assert size(4096, 100, 64, 16, 8, 128) >= 2 * 64 * 16 * 128 * 4
    assert size(4096, 100, 0, 16, 8, 128) == 0 and size(4096, 100, 4, 16, 0, 128) == 0


def test_binding_refuses_tensors_that_do_not_fit(built_lib):
    """Shapes, types and devices, before the library is called: CPU tensors reach the device check last."""
    import torch

    from funasrnet_b200 import device_ops

    native = device_ops._native()
    q, k = torch.zeros(7, 4, 64, dtype=torch.half), torch.zeros(9, 2, 64, dtype=torch.half)
    off = torch.zeros(3, dtype=torch.int32)

    def go(q=q, k=k, v=k, qo=off, ko=off, out=q, scale=None, lse=None, workspace=None, stream=None):
        return native.attention_packed(0, 0, q, k, v, qo, ko, out, True, scale, lse, workspace, stream)

    for kw, word in ((dict(), "not on the backend's device"), (dict(q=7), "expected a torch tensor"),
                     (dict(q=q[0]), "three dimensions"), (dict(q=q.double()), "expected float32"),
                     (dict(k=k[..., :32]), "head size"), (dict(qo=off[:0]), "empty")):
        with pytest.raises(ValueError, match=word):
            go(**kw)
    with pytest.raises(TypeError):
        native.attention_packed(0, 0, q)
    x = torch.zeros(3, 100)
    none = [None] * 13
    with pytest.raises(ValueError, match="not on the backend's device"):
        native.adjust_logits(0, 0, x, x, *none)
    with pytest.raises(ValueError, match="two dimensions"):
        native.adjust_logits(0, 0, x[0], x, *none)
    with pytest.raises(ValueError, match="expected a torch tensor"):
        native.attention_shared(0, 0, q, k, k, None, k, off, q, None, None, None, None)


def test_the_backends_stream_needs_a_backend(built_lib):
    from funasrnet_b200._lib import lib

    out = C.c_void_p()
    assert lib().fa_backend_stream(None, C.byref(out)) == ARGUMENT


def test_binding_refuses_tensors_that_require_grad(built_lib):
    """Wherever such a tensor stands, before anything else is looked at; under no_grad it is taken."""
    import torch

    from funasrnet_b200 import device_ops

    native = device_ops._native()
    half, off = torch.zeros(7, 4, 64, dtype=torch.half), torch.zeros(2, dtype=torch.int32)
    cache = torch.zeros(7, 9, 4, 64, dtype=torch.half)
    packed = [0, 0, half, half, half, off, off, half, True, None, None, None, None]
    shared = [0, 0, half, half, half, cache, cache, torch.zeros(7, dtype=torch.int32), half, None, None, None, None]
    x, f = torch.zeros(3, 100), torch.zeros(3)
    logits = [0, 0, x, x, None, None, None, None, f, f, f, None, None, None, None, None, None]
    for fn, args, places in ((native.attention_packed, packed, (2, 3, 4, 7)), (native.attention_shared, shared, (2, 3, 4, 5, 6, 8)),
                             (native.adjust_logits, logits, (2, 3, 8, 9, 10))):
        with pytest.raises(ValueError, match="not on the backend's device"):
            fn(*args)
        for i in places:
            with_grad = args[:i] + [args[i].clone().requires_grad_()] + args[i + 1:]
            with pytest.raises(ValueError, match="requires grad"):
                fn(*with_grad)
            with torch.no_grad(), pytest.raises(ValueError, match="not on the backend's device"):
                fn(*with_grad)


def test_workspace_bounds_hold_for_every_smaller_call(built_lib):
    """Sizes that grow when a batch shrinks, then random ones: no call up to the given sizes needs more than their bound,
    and bounds grow with the sizes."""
    import random

    from funasrnet_b200._lib import lib

    packed_size, packed_bound = lib().fa_dev_attention_packed_workspace, lib().fa_dev_attention_packed_workspace_bound
    shared_size, shared_bound = lib().fa_dev_attention_shared_workspace, lib().fa_dev_attention_shared_workspace_bound
    assert packed_size(300, 1000, 1, 16, 8, 128) < packed_size(100, 1000, 1, 16, 8, 128) <= packed_bound(300, 1000, 16, 8, 128)
    assert shared_size(2048, 4000, 4, 16, 8, 128) < shared_size(2048, 4000, 3, 16, 8, 128)
    assert shared_size(2048, 4000, 3, 16, 8, 128) <= shared_bound(2048, 4000, 4, 16, 8, 128)
    assert shared_size(2048, 100, 85, 16, 8, 128) <= shared_bound(2048, 100, 86, 16, 8, 128)
    rng = random.Random(17)

    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    for _ in range(4000):
        kv_heads, group, head = rng.choice([1, 2, 8, 16]), rng.choice([1, 2, 3, 7, 8, 64]), rng.choice([8, 64, 72, 128])
        heads = kv_heads * group
        q, k = size(1, 60000), size(1, 1 << 22)
        bound = packed_bound(q, k, heads, kv_heads, head)
        assert bound <= packed_bound(2 * q, k, heads, kv_heads, head) and bound <= packed_bound(q, 3 * k, heads, kv_heads, head)
        for _ in range(25):
            assert packed_size(size(1, q), size(1, k), size(1, 200), heads, kv_heads, head) <= bound
        prefix, cap, n = size(1, 300000) - 1, size(1, 20000) - 1, size(1, 600)
        bound = shared_bound(prefix, cap, n, heads, kv_heads, head)
        for bigger in ((2 * prefix, cap, n), (prefix, 2 * cap, n), (prefix, cap, 2 * n)):
            assert bound <= shared_bound(*bigger, heads, kv_heads, head)
        for _ in range(25):
            assert shared_size(size(1, prefix + 1) - 1, size(1, cap + 1) - 1, size(1, n), heads, kv_heads, head) <= bound
        assert shared_size(prefix, cap, n, heads, kv_heads, head) <= bound
    # Nothing to cut, sizes out of range, and the largest.
    assert packed_bound(100, 511, 16, 8, 128) == 0 and shared_bound(0, 300, 500, 16, 8, 128) == 0
    assert packed_bound(-1, 5, 8, 8, 128) == packed_bound(5, 5, 15, 8, 128) == shared_bound(5, 5, 0, 8, 8, 128) == 0
    assert 0 < packed_bound(1 << 62, 1 << 62, 16, 8, 128) < 1 << 30
    assert 0 < shared_bound((1 << 63) - 1, (1 << 63) - 1, 100, 16, 8, 128) < 1 << 30
    assert shared_bound(1 << 40, 1 << 40, (1 << 31) - 1, (1 << 31) - 1, (1 << 31) - 1, 128) > 0


@pytest.mark.parametrize("make,change", [
    (packed, dict(lse=66)),
    (packed, dict(q_offsets=65)),
    (packed, dict(k_offsets=62)),
    (shared, dict(lse=2)),
    (shared, dict(suffix_lens=67)),
    (logits, dict(logits=(1 << 20) + 2)),
    (logits, dict(out=(1 << 22) + 1)),
    (logits, dict(dtype=BF16, logits=(1 << 20) + 1)),
    (logits, dict(tokens=65)),
    (logits, dict(history=66, history_offsets=64)),
    (logits, dict(history=64, history_offsets=66)),
    (logits, dict(prompt_lens=66)),
    (logits, dict(repetition=66)),
    (logits, dict(presence=66)),
    (logits, dict(frequency=66)),
    (logits, dict(bias_tokens=66, bias_values=64, bias_offsets=64)),
    (logits, dict(bias_tokens=64, bias_values=66, bias_offsets=64)),
    (logits, dict(bias_tokens=64, bias_values=64, bias_offsets=66)),
    (logits, dict(mask=66, mask_count=4, mask_stride=32)),
    (logits, dict(mask_rows=66)),
])
def test_addresses_off_their_types_are_refused(call, make, change):
    """The device would fault on them."""
    rc, message = call(make(**change))
    assert rc == ARGUMENT and "aligned" in message, message


def test_half_rows_on_two_bytes_are_taken(call):
    assert call(logits(dtype=F16, logits=(1 << 20) + 2, out=(1 << 22) + 6)) == (ARGUMENT, "null backend")


@pytest.mark.parametrize("make,change", [
    (packed, dict(total_q=(1 << 31) - 100, total_k=50, heads=1, kv_heads=1)),
    (packed, dict(total_q=(1 << 31) - (1 << 20), total_k=1 << 20, heads=1, kv_heads=1)),
    (shared, dict(sequences=(1 << 31) - 100, heads=1, kv_heads=1)),
])
def test_sizes_whose_sums_pass_32_bits_are_declined(call, make, change):
    """The kernels add a tile's rows to a token, and keys to tokens, in 32 bits."""
    assert call(make(**change))[0] == DECLINED


def test_the_largest_sums_are_taken(call):
    change = dict(total_q=(1 << 31) - (1 << 20), total_k=(1 << 20) - 1024, heads=1, kv_heads=1)
    assert call(packed(**change)) == (ARGUMENT, "null backend")
