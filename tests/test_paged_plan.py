"""The paged attention's plan on the CPU: its units cover every query row and
every key that the row sees exactly once, parts of an item agree with one another
and own scratch rows and counters of their own, work is spread evenly, and what a
plan or a wrapper cannot take is refused with a reason."""
import random

import pytest
import torch

from emmy_b200 import native, paged

pytestmark = pytest.mark.usefixtures("native_lib")

FIELDS = ("seq", "kvh", "tok0", "ntok", "pos0", "tile0", "ntiles", "lo", "hi", "kv_len", "wide", "item", "split",
          "nsplit", "part_row", "pad")


def units_of(plan):
    w = plan.words.tolist()
    ctas, counters, at = w[1:4]
    first = w[4:4 + ctas + 1]
    units = [dict(zip(FIELDS, w[at + 16 * i:at + 16 * i + 16])) for i in range(first[-1])]
    assert len(w) == at + 16 * len(units) and at % 16 == 0 and w[0] == 0
    assert all(x == 0 for x in w[counters:at])
    assert first[0] == 0 and all(a < b for a, b in zip(first, first[1:]))
    return units, first, (at - counters) // 2


CASES = [
    ([1], [301], 32, 8, True, 0),
    ([1], [131071], 32, 8, True, 0),
    ([1] * 64, [random.Random(s).randint(1, 8191) for s in range(64)], 32, 8, True, 0),
    ([4096] * 4, [4096] * 4, 32, 8, True, 0),
    ([1, 511, 1, 77, 0, 300], [5000, 12288, 0, 77, 900, 299], 32, 4, True, 0),
    ([1501, 2048], [4097, 8192], 32, 8, True, 1024),
    ([9, 2, 64], [20, 2, 640], 6, 2, True, 5),
    ([33], [1000], 40, 8, False, 0),
    ([128], [16384], 128, 1, True, 0),
    ([700], [65536], 5, 1, True, 0),
    ([0, 0], [10, 0], 4, 4, True, 0),
    ([], [], 4, 4, True, 0),
]


@pytest.mark.parametrize("q_lens,kv_lens,hq,hkv,causal,window", CASES)
@pytest.mark.parametrize("ctas", [1, 7, 148])
def test_units_cover_the_work_once(q_lens, kv_lens, hq, hkv, causal, window, ctas):
    plan = paged.AttentionPlan(q_lens, kv_lens, hq, hkv, 64, causal, window or None, device="cpu", ctas=ctas)
    if not sum(q_lens):
        assert len(units_of(plan)[0]) == 0
        return
    units, first, counters = units_of(plan)
    group = hq // hkv
    per_tile = 128 // group
    start = [sum(q_lens[:s]) for s in range(len(q_lens))]
    items = {}
    for u in units:
        assert 0 < u["ntok"] <= 2 * per_tile and u["wide"] == (u["ntok"] > per_tile)
        items.setdefault((u["seq"], u["kvh"], u["tok0"]), []).append(u)
    rows, scratch, numbers = {}, set(), set()
    for (s, h, tok0), us in items.items():
        t0 = tok0 - start[s]
        assert 0 <= t0 and t0 + us[0]["ntok"] <= q_lens[s] and 0 <= h < hkv
        for t in range(us[0]["ntok"]):
            assert (tok0 + t, h) not in rows
            rows[tok0 + t, h] = True
        # the keys the block's tokens see between them
        seen = []
        for t in (t0, t0 + us[0]["ntok"] - 1):
            pos = kv_lens[s] - q_lens[s] + t
            seen += [max(0, pos - window + 1) if window else 0, min(kv_lens[s], pos + 1) if causal else kv_lens[s]]
        lo, hi = seen[0], seen[3]
        tiles = sorted((u["tile0"], u["ntiles"], u["split"]) for u in us)
        if hi <= lo:
            assert [u["ntiles"] for u in us] == [0]
        else:
            at = lo // 128
            for k, (tile0, n, split) in enumerate(tiles):
                assert tile0 == at and n > 0 and split == k
                at += n
            assert at == -(-hi // 128)
            assert (us[0]["lo"], us[0]["hi"]) == (lo, hi)
        assert all(u["nsplit"] == len(us) for u in us)
        assert len({(u["item"], u["part_row"], u["pos0"], u["kv_len"]) for u in us}) == 1
        assert us[0]["pos0"] == kv_lens[s] - q_lens[s] + t0
        if len(us) > 1:
            assert us[0]["item"] < counters and us[0]["item"] not in numbers
            numbers.add(us[0]["item"])
            mine = set(range(us[0]["part_row"], us[0]["part_row"] + len(us) * us[0]["ntok"] * group))
            assert not mine & scratch
            scratch |= mine
    assert len(rows) == sum(q_lens) * hkv
    assert plan.scratch.numel() == len(scratch) * (64 + 2) * 4
    assert not scratch or max(scratch) + 1 == len(scratch)


@pytest.mark.parametrize("q_lens,kv_lens,most", [
    ([1] * 64, [random.Random(s).randint(517, 8191) for s in range(64)], 1.03),
    ([1], [131071], 1.1),
    ([4096] * 8, [4096] * 8, 1.05),
])
def test_work_is_even(q_lens, kv_lens, most):
    plan = paged.AttentionPlan(q_lens, kv_lens, 32, 8, 128, device="cpu", ctas=148)
    units, first, _ = units_of(plan)
    load = [sum(u["ntiles"] for u in units[a:b]) for a, b in zip(first, first[1:])]
    assert max(load) <= most * sum(load) / 148 + 2, (max(load), sum(load) / 148)


@pytest.mark.parametrize("change,words", [
    (dict(q_heads=33), "query heads"), (dict(kv_heads=0), "query heads"), (dict(q_heads=8 * 129), "query heads"),
    (dict(head_dim=96), "head_dim"), (dict(causal=False, window=4), "window"), (dict(ctas=0), "CTAs"),
])
def test_plan_refuses(change, words):
    a = dict(q_lens=[1], kv_lens=[5], q_heads=32, kv_heads=8, head_dim=128, device="cpu", ctas=148) | change
    with pytest.raises(native.EmmyError, match=words) as e:
        paged.AttentionPlan(**a)
    assert e.value.code == -1


@pytest.mark.parametrize("change", [dict(q_lens=[1, 2]), dict(q_lens=[-1]), dict(window=0), dict(kv_lens=[1 << 31])])
def test_wrapper_refuses(change):
    a = dict(q_lens=[1], kv_lens=[5], q_heads=32, kv_heads=8, head_dim=128, device="cpu", ctas=148) | change
    with pytest.raises(ValueError):
        paged.AttentionPlan(**a)


def test_operators_need_cuda_tensors():
    t = torch.zeros(1, 8, 64)
    with pytest.raises(ValueError, match="CUDA"):
        paged.rotate_append(None, t, t, t, None, None, None, None)
    plan = paged.AttentionPlan([1], [5], 8, 8, 64, device="cpu", ctas=1)
    with pytest.raises(ValueError, match="CUDA"):
        paged.attention(plan, t, None, None, None)


def _rotate_args(**change):
    names = ("dtype", "tokens", "q_heads", "kv_heads", "head_dim", "rotary_dim", "axes", "interleaved", "pages", "page_size",
             "q", "k", "v", "q_out", "k_cache", "v_cache", "positions", "slots", "frequencies", "pair_axis")
    a = dict(zip(names, [9, 3, 4, 2, 64, 64, 1, 0, 8, 16] + [4096] * 9 + [0])) | change
    return paged._ROTATE_APPEND_ARGS.pack(*a.values(), 256, 64, 128, 64, 128, 64, 256, 64, 2048, 128, 64, 2048, 128, 64, 3)


@pytest.mark.parametrize("change,words", [
    (dict(dtype=10), b"dtype"), (dict(tokens=-1), b"count"), (dict(q_heads=-1), b"count"), (dict(head_dim=0), b"head_dim"),
    (dict(head_dim=257), b"head_dim"), (dict(rotary_dim=65), b"rotary_dim"), (dict(rotary_dim=66), b"rotary_dim"),
    (dict(axes=0), b"axes"), (dict(page_size=0), b"cache"), (dict(q=0), b"null"), (dict(slots=0), b"null"),
    (dict(positions=0), b"null"), (dict(v_cache=0), b"null"), (dict(k=4097), b"multiple"), (dict(frequencies=4098), b"multiple"),
])
def test_c_rotate_append_refuses(native_lib, change, words):
    """Refused before anything of CUDA is called: no GPU is needed."""
    assert native_lib.emmy_rotate_append(_rotate_args(**change), None) == -1
    assert words in native_lib.emmy_last_error()


def test_c_null_arguments(native_lib):
    assert native_lib.emmy_rotate_append(None, None) == -1
    assert native_lib.emmy_paged_plan_make(None, None) == -1
    assert native_lib.emmy_paged_plan_data(None, None, None, None) == -1
    assert native_lib.emmy_paged_attention(None, None, None) == -1
    assert native_lib.emmy_paged_plan_status(None, 0, None) == -1
    native_lib.emmy_paged_plan_free(None)
    assert native_lib.emmy_rotate_append(_rotate_args(tokens=0), None) == 0


@pytest.mark.parametrize("change,words", [
    (dict(dtype=7), b"dtype"), (dict(scale=-1.0), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(page_size=24), b"page_size"),
    (dict(page_size=192), b"page_size"), (dict(pages=0), b"pages"), (dict(table_width=1), b"does not hold"), (dict(q=0), b"null"),
    (dict(scratch=0), b"null"), (dict(q=4104), b"16 bytes"), (dict(scratch=4112), b"16 bytes"), (dict(table=4098), b"16 bytes"),
    (dict(q_token=100), b"stride"), (dict(k_page=-2048), b"stride"), (dict(v_token=0), b"stride"),
])
def test_c_attention_refuses(native_lib, change, words):
    plan = paged.AttentionPlan([2], [5000], 8, 2, 64, device="cpu", ctas=148)
    assert plan.scratch.numel()
    names = ("dtype", "pages", "page_size", "table_width", "scale", "q", "out", "lse", "k_cache", "v_cache", "table",
             "plan_words", "scratch", "q_token", "q_head", "out_token", "out_head", "k_page", "k_token", "k_head",
             "v_page", "v_token", "v_head", "table_stride")
    a = dict(zip(names, [9, 400, 16, 400, 0.125] + [4096] * 8 + [512, 64, 512, 64, 2048, 128, 64, 2048, 128, 64, 400])) | change
    assert native_lib.emmy_paged_attention(plan._h, paged._ATTENTION_ARGS.pack(*a.values()), None) == -1
    assert words in native_lib.emmy_last_error(), native_lib.emmy_last_error()
