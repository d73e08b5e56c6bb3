"""Paged-cache operators on the CPU: arguments at the ends of their ranges, and the
order and streams that the kernels and their memory rely on."""
import random
import sys

import pytest
import torch

from emmy_b200 import native, paged
from test_paged_plan import units_of

pytestmark = pytest.mark.usefixtures("native_lib")


# --------------------------------------------------------------------- windows
def c_plan_words(q_lens, kv_lens, window):
    """Words of a plan made through the C ABI, where a window has 32 bits."""
    import ctypes
    lens = (ctypes.c_int32 * (2 * len(q_lens)))(*q_lens, *kv_lens)
    a = paged._PlanArgs(len(q_lens), ctypes.addressof(lens), ctypes.addressof(lens) + 4 * len(q_lens), 8, 2, 64, 1, window, 148)
    L, h = native.lib(), ctypes.c_void_p()
    native.check(L.emmy_paged_plan_make(ctypes.byref(a), ctypes.byref(h)))
    words, count, scratch = ctypes.c_void_p(), ctypes.c_size_t(), ctypes.c_size_t()
    native.check(L.emmy_paged_plan_data(h, ctypes.byref(words), ctypes.byref(count), ctypes.byref(scratch)))
    got = list((ctypes.c_int32 * count.value).from_address(words.value))
    L.emmy_paged_plan_free(h)
    return got


LENGTHS = [([10], [4]), ([40, 1], [30, 1000]), ([1], [1]), ([2 ** 20], [0]), ([300, 7], [5000, 2])]


@pytest.mark.parametrize("q_lens,kv_lens", LENGTHS)
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30])
def test_windows_of_31_bits_hide_nothing(q_lens, kv_lens, window):
    assert c_plan_words(q_lens, kv_lens, window) == c_plan_words(q_lens, kv_lens, 0)


@pytest.mark.parametrize("q_lens,kv_lens", LENGTHS)
@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, sys.maxsize, 2 ** 64])
def test_windows_beyond_every_length(q_lens, kv_lens, window):
    plans = [paged.AttentionPlan(q_lens, kv_lens, 8, 2, 64, window=w, device="cpu", ctas=148) for w in (window, None)]
    assert plans[0].words.tolist() == plans[1].words.tolist()


def test_the_longest_window_that_hides_a_key():
    """One position less than the longest sequence has: its last token does not see the first."""
    plan = paged.AttentionPlan([1, 1], [100, 1000], 8, 2, 64, window=999, device="cpu", ctas=148)
    assert {(u["seq"], u["lo"]) for u in units_of(plan)[0]} == {(0, 0), (1, 1)}


# --------------------------------------------------------------------- numbers
@pytest.mark.parametrize("change", [dict(q_heads=2 ** 32 + 32), dict(kv_heads=2 ** 32 + 8), dict(head_dim=2 ** 32 + 128), dict(ctas=2 ** 32 + 1),
                                    dict(ctas=-2 ** 32 + 1), dict(q_heads=2 ** 31)])
def test_counts_beyond_32_bits_are_refused(change):
    """Not taken as their lowest 32 bits."""
    a = dict(q_lens=[1], kv_lens=[5], q_heads=32, kv_heads=8, head_dim=128, device="cpu", ctas=148) | change
    with pytest.raises(ValueError, match="32 bits"):
        paged.AttentionPlan(**a)


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_c_attention_refuses_scales_without_a_base_of_2(native_lib, scale):
    """scale x log2(e) has to be finite as well."""
    plan = paged.AttentionPlan([2], [5000], 8, 2, 64, device="cpu", ctas=148)
    a = paged._ATTENTION_ARGS.pack(9, 400, 16, 400, scale, *[4096] * 8, 512, 64, 512, 64, 2048, 128, 64, 2048, 128, 64, 400)
    assert native_lib.emmy_paged_attention(plan._h, a, None) == -1
    assert b"scale" in native_lib.emmy_last_error(), native_lib.emmy_last_error()


# ------------------------------------------------------------- nothing to read
@pytest.mark.parametrize("change", [dict(table=0, table_width=0), dict(pages=0, k_cache=0, v_cache=0), dict(pages=0, table=0, table_width=0)])
@pytest.mark.parametrize("kv_lens,refused", [([0, 0], False), ([0, 1], True), ([3, 0], True)])
def test_a_cache_is_needed_where_a_token_sees_a_key(native_lib, change, kv_lens, refused):
    """Refused for its arguments (before any CUDA call), or not."""
    plan = paged.AttentionPlan([2, 3], kv_lens, 8, 2, 64, causal=False, device="cpu", ctas=148)
    names = ("dtype", "pages", "page_size", "table_width", "scale", "q", "out", "lse", "k_cache", "v_cache", "table")
    a = dict(zip(names, [9, 400, 16, 400, 0.125] + [4096] * 6)) | change
    a = paged._ATTENTION_ARGS.pack(*a.values(), 4096, 4096, 512, 64, 512, 64, 2048, 128, 64, 2048, 128, 64, 400)
    if not refused and torch.cuda.is_available():
        pytest.skip("would run")
    native_lib.emmy_paged_attention(plan._h, a, None)
    said = any(word in native_lib.emmy_last_error() for word in (b"null", b"does not hold", b"a cache of"))
    assert said == refused, native_lib.emmy_last_error()


# --------------------------------------------------------------------- streams
@pytest.mark.parametrize("handle,name", [(0, "default"), (1, "default"), (2, "external 2"), (4096, "external 4096")])
def test_memory_is_recorded_on_the_stream_that_a_handle_names(monkeypatch, handle, name):
    """0 and 1 are the default stream; as an external one, 0 would be a stream of PyTorch's own."""
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda at, device=None: f"external {at}")
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: "default")
    recorded = []

    class Memory:
        device = torch.device("cuda", 0)
        record_stream = recorded.append

    paged._made_for(handle, Memory())
    assert recorded == [name]


def test_memory_that_others_allocated_is_recorded_on_every_stream(monkeypatch):
    """Also on the stream that was current when it was handed over: it need not be from there."""
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 4096, raising=False)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda at, device=None: at)
    recorded = []

    class Memory:
        device = torch.device("cuda", 0)
        record_stream = recorded.append

    kept = paged._Kept()
    kept._keep(Memory(), None)
    for stream in (4096, 8192, 4096, 8192):
        if stream not in kept._streams:
            kept._used_on(stream)
    assert recorded == [4096, 8192]


@pytest.mark.parametrize("used,given,waits", [({7}, None, False), ({8}, None, True), ({7, 8}, None, True), (set(), None, False),
                                              ({7, 8}, 8, False)])
def test_check_waits_for_every_stream_that_calls_ran_on(monkeypatch, used, given, waits):
    """On the current one (7) alone its status is read in order; others are waited for first."""
    plan = paged.AttentionPlan([1], [5], 8, 8, 64, device="cpu", ctas=1)
    did = []
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 7, raising=False)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: did.append("all"))
    monkeypatch.setattr(paged, "_call", lambda name, index, stream, *args: did.append(stream))
    plan._streams = used
    plan.check(given)
    assert did == ["all"] * waits + [given or 7]


# ----------------------------------------------------------------------- order
@pytest.mark.parametrize("seed", range(40))
def test_wide_units_of_a_cta_come_first(seed):
    """The kernel gives what a unit of few rows joins the place of a wide unit's queries."""
    r = random.Random(seed)
    n = r.randint(1, 12)
    q_lens = [r.choice((0, 1, 1, 2, 17, 64, 300, 1000)) for _ in range(n)]
    kv_lens = [r.choice((0, 5, 130, 1000, 9000)) for _ in range(n)]
    kv_heads = r.choice((1, 2, 8))
    plan = paged.AttentionPlan(q_lens, kv_lens, kv_heads * r.choice((1, 3, 4, 32)), kv_heads, r.choice((64, 128)),
                               window=r.choice((None, 100)), device="cpu", ctas=r.choice((1, 2, 7, 148)))
    units, first, _ = units_of(plan)
    for a, b in zip(first, first[1:]):
        wide = [u["wide"] for u in units[a:b]]
        assert wide == sorted(wide, reverse=True)
