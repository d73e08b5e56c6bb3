"""The plan of attention over an 8-bit cache on the CPU: its pieces and read-back jobs
cover every query row and every key that the row sees exactly once, parts own scratch
rows and counters of their own, work is even, and what the operators of an 8-bit cache
and of drafted tokens cannot take is refused before any CUDA call."""
import random

import pytest
import torch

from emmy_b200 import native, paged

pytestmark = pytest.mark.usefixtures("native_lib")

FIELDS = ("seq", "kvh", "tok0", "row0", "rows", "pos0", "lo", "hi", "kv_len", "slice0", "nslices", "split", "nsplit", "part_row")
FEW, MIDDLE = 24, 128                 # rows of 64 components


def parts_of(plan):
    """(pieces, where the lists of each CTA and warp begin, warps)"""
    w = plan.words.tolist()
    ctas, warps, at, status = w[:4]
    first = w[4:4 + ctas * (warps + 1) + 1]
    assert status == 0 and first[0] == 0 and all(a <= b for a, b in zip(first, first[1:])) and at % 16 == 0
    assert not any(w[4 + len(first):at])
    return [dict(zip(FIELDS, w[at + 16 * i:at + 16 * i + 14])) for i in range(first[-1])], first, warps


def rows_to_join(plan, pieces, group):
    """Behind the pieces: (part_row, step, nsplit, token, head) of each row of an item of several parts."""
    w, at = plan.words.tolist(), plan.words.tolist()[2] + 16 * len(pieces)
    n = sum(u["rows"] for u in pieces if u["nsplit"] > 1 and u["split"] == 0)
    return [tuple(w[at + 8 * i:at + 8 * i + 5]) for i in range(n)]


CASES = [
    ([1], [301], 32, 8, True, 0),
    ([1], [131071], 32, 8, True, 0),
    ([1] * 64, [random.Random(s).randint(1, 8191) for s in range(64)], 32, 8, True, 0),
    ([3, 9, 0, 30, 1], [3000, 12288, 0, 77, 900], 32, 8, True, 0),
    ([9, 2, 64], [20, 2, 640], 6, 2, True, 5),
    ([33], [1000], 40, 8, False, 0),
    ([1], [16384], 128, 1, True, 0),
    ([2, 5], [9, 2], 4, 4, True, 0),
    ([7, 25], [65536, 5000], 5, 1, True, 333),
    ([500, 1, 300], [700, 9000, 200], 8, 2, True, 0),
    ([0, 0], [10, 0], 4, 4, True, 0),
    ([4], [100], 127, 1, True, 0),
    ([5], [100], 127, 1, True, 0),
    ([9, 1], [100, 90], 100, 1, True, 0),
    ([], [], 4, 4, True, 0),
]


@pytest.mark.parametrize("q_lens,kv_lens,hq,hkv,causal,window", CASES)
@pytest.mark.parametrize("ctas", [1, 7, 148])
def test_pieces_cover_the_work_once(q_lens, kv_lens, hq, hkv, causal, window, ctas):
    plan = paged.QuantisedPlan(q_lens, kv_lens, hq, hkv, 64, causal, window or None, device="cpu", ctas=ctas)
    pieces, first, warps = parts_of(plan)
    group = hq // hkv
    kinds = [0 if q * group <= FEW else 1 if q * group <= MIDDLE else 2 for q in q_lens]
    # (all are few where that is not much, or the middle ones where there are no others)
    more = [(kv if not window else min(kv, window + q), -(-q * group // 16)) for q, kv, k in zip(q_lens, kv_lens, kinds) if k and q]
    if all(q * group * group < 2 ** 15 for q, k in zip(q_lens, kinds) if k) and sum(b for _, b in more) * hkv <= 2 * ctas and len(more) * hkv * sum(n * b for n, b in more) * hkv * 64 ** 2 <= 2 ** 36:
        kinds = [0] * len(kinds)
    # (few and middle ones of little go with those that are read back)
    seen = [min(kv, window + q if window else kv) * hkv * 64 * 2 if q else 0 for q, kv in zip(q_lens, kv_lens)]
    small = 0
    for k in (1, 0):
        mine = sum(b for b, kind in zip(seen, kinds) if kind == k)
        if mine and any(b for b, kind in zip(seen, kinds) if kind == 2) and small + mine <= 2 ** 25:
            small += mine
            kinds = [2 if kind == k and q else kind for kind, q in zip(kinds, q_lens)]
    few = [k == 0 for k in kinds]
    at_once = {8: 8, 6: 16}[warps]
    assert len(first) - 1 <= 2 * ctas * (warps + 1)
    items = {}
    for u in pieces:
        assert few[u["seq"]] and 0 < u["rows"] <= at_once and 0 <= u["kvh"] < hkv
        assert u["tok0"] == sum(q_lens[:u["seq"]]) and u["pos0"] == kv_lens[u["seq"]] - q_lens[u["seq"]] and u["kv_len"] == kv_lens[u["seq"]]
        items.setdefault((u["seq"], u["kvh"], u["row0"]), []).append(u)
    covered, scratch, joined = set(), set(), set()
    for (s, h, row0), us in items.items():
        rows = range(row0, row0 + us[0]["rows"])
        assert rows.stop <= q_lens[s] * group
        mine = {(s, h, r) for r in rows}
        assert not mine & covered
        covered |= mine
        lows = [max(0, us[0]["pos0"] + r // group - window + 1) if window else 0 for r in rows]
        highs = [min(kv_lens[s], us[0]["pos0"] + r // group + 1) if causal else kv_lens[s] for r in rows]
        lo, hi = min(lows), max(highs + [0])
        if hi <= lo:
            assert [u["nslices"] for u in us] == [0]
        else:
            at = lo // 32                # slices of 32 keys of 64 components
            for k, u in enumerate(sorted(us, key=lambda u: u["split"])):
                assert (u["slice0"], u["split"], u["lo"], u["hi"]) == (at, k, lo, hi) and u["nslices"] > 0
                at += u["nslices"]
            assert at == -(-hi // 32)
        assert all((u["nsplit"], u["part_row"], u["rows"]) == (len(us), us[0]["part_row"], us[0]["rows"]) for u in us)
        if len(us) > 1:
            joined |= {(us[0]["part_row"] + r - row0, len(rows), len(us), us[0]["tok0"] + r // group, h * group + r % group) for r in rows}
            mine = set(range(us[0]["part_row"], us[0]["part_row"] + len(us) * us[0]["rows"]))
            assert not mine & scratch
            scratch |= mine
    assert len(covered) == sum(q * hq for q, f in zip(q_lens, few) if f)
    assert scratch == set(range(len(scratch))) and joined == set(rows_to_join(plan, pieces, group))
    # keys that are read back: 4 bytes a component of whole pages of 128 tokens that some row sees; and parts
    blocks = 0
    for q, kv, kind in zip(q_lens, kv_lens, kinds):
        hi, lo = kv, max(0, kv - q - window + 1) if window else 0
        blocks += -(-hi // 128) - lo // 128 if kind == 2 and hi > 0 else 0
    assert plan.scratch.numel() >= len(scratch) * 68 * 4 + blocks * 128 * hkv * 64 * 4
    if all(few):
        assert plan.scratch.numel() == -(-len(scratch) * 68 * 4 // 128) * 128


@pytest.mark.parametrize("q_lens,kv_lens,most", [
    ([1] * 64, [random.Random(s).randint(517, 8191) for s in range(64)], 1.03),
    ([1], [131071], 1.03),
    ([4] * 24, [random.Random(s).randint(65, 4095) for s in range(24)], 1.2),
])
def test_work_is_even(q_lens, kv_lens, most):
    plan = paged.QuantisedPlan(q_lens, kv_lens, 32, 8, 128, device="cpu", ctas=148)
    pieces, first, warps = parts_of(plan)
    load = []
    for c in range(0, len(first) - 1, warps + 1):
        shared, *own = (sum(u["nslices"] for u in pieces[a:b]) for a, b in zip(first[c:], first[c + 1:c + warps + 2]))
        load.append(-(-shared // warps) + max(own))
    even = sum(u["nslices"] for u in pieces) / 296 / warps
    assert max(load) <= most * even + 4, (max(load), even)


def test_rows_of_a_piece_can_be_divided():
    """The kernel for few rows takes row * ceil(2^16 / G) >> 16 for row / G: right for every row that it is given."""
    for group in range(1, 129):
        most = max(24, (2 ** 15 - 1) // group)
        inverse = -(-2 ** 16 // group)
        assert most * inverse < 2 ** 31 and all(r * inverse >> 16 == r // group for r in range(most + 1)), group


@pytest.mark.parametrize("seed", range(30))
def test_parts_of_random_plans(seed):
    """Whatever is shared or a warp's own: each item's slices once, in order of its parts."""
    r = random.Random(seed)
    n, kv_heads, group = r.randint(1, 70), r.choice((1, 2, 3, 4, 6, 8, 32)), r.choice((1, 2, 4, 5, 8, 16))
    q_lens = [r.choice((1, 1, 1, r.randint(0, 9), r.randint(0, 40))) for _ in range(n)]
    kv_lens = [r.choice((0, r.randint(1, 300), r.randint(1, 9000))) for _ in range(n)]
    test_pieces_cover_the_work_once(q_lens, kv_lens, group * kv_heads, kv_heads, r.random() < 0.8, 0, r.choice((1, 5, 148)))


@pytest.mark.parametrize("change,words", [
    (dict(q_heads=33), "query heads"), (dict(kv_heads=0), "query heads"), (dict(q_heads=8 * 129), "query heads"),
    (dict(head_dim=96), "head_dim"), (dict(causal=False, window=4), "window"), (dict(ctas=0), "CTAs"),
])
def test_plan_refuses(change, words):
    a = dict(q_lens=[1], kv_lens=[5], q_heads=32, kv_heads=8, head_dim=128, device="cpu", ctas=148) | change
    with pytest.raises(native.EmmyError, match=words) as e:
        paged.QuantisedPlan(**a)
    assert e.value.code == -1


@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31, 2 ** 64, 1000])
def test_windows_beyond_every_length(window):
    plans = [paged.QuantisedPlan([1, 200], [999, 1000], 8, 2, 64, window=w, device="cpu", ctas=148) for w in (window, None)]
    assert plans[0].words.tolist() == plans[1].words.tolist()


def test_plans_of_one_operator_are_not_the_others():
    q = torch.zeros(1, 8, 64)
    for plan, call in ((paged.AttentionPlan, paged.quantised_attention),):
        with pytest.raises(ValueError, match="QuantisedPlan"):
            call(plan([1], [5], 8, 8, 64, device="cpu", ctas=1), q, q, q, None, q)


def test_operators_need_cuda_tensors():
    t = torch.zeros(1, 8, 64)
    with pytest.raises(ValueError, match="CUDA"):
        paged.norm_rotate_append(None, None, t, t, t, None, None, None, None)
    with pytest.raises(ValueError, match="CUDA"):
        paged.quantised_attention(paged.QuantisedPlan([1], [5], 8, 8, 64, device="cpu", ctas=1), t, None, None, None, None)
    with pytest.raises(ValueError, match="CUDA"):
        paged.verify(t[0], None, None, None, None, None)
    with pytest.raises(ValueError, match="CUDA"):
        paged.Norm(t[0, 0], t[0, 0])


def test_c_null_arguments(native_lib):
    assert native_lib.emmy_norm_rotate_append(None, None) == -1
    assert native_lib.emmy_quantised_plan_make(None, None) == -1
    assert native_lib.emmy_quantised_plan_data(None, None, None, None) == -1
    assert native_lib.emmy_quantised_attention(None, None, None) == -1
    assert native_lib.emmy_quantised_plan_status(None, 0, None) == -1
    assert native_lib.emmy_verify(None, None) == -1
    native_lib.emmy_quantised_plan_free(None)


@pytest.mark.parametrize("change,words", [
    (dict(dtype=10), b"dtype"), (dict(tokens=-1), b"count"), (dict(head_dim=257), b"head_dim"), (dict(rotary_dim=65), b"rotary_dim"),
    (dict(axes=0), b"axes"), (dict(page_size=0), b"cache"), (dict(q=0), b"null"), (dict(v_cache=0), b"null"), (dict(k=4097), b"multiple"),
    (dict(q_weight=0), b"null"), (dict(k_weight=0), b"null"), (dict(k_weight=4097), b"multiple"), (dict(exponents=4098), b"multiple"),
    (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(bits8=2), b"cache_bits8"), (dict(bits8=0, k_cache=4097), b"multiple"),
])
def test_c_norm_rotate_append_refuses(native_lib, change, words):
    names = ("dtype", "tokens", "q_heads", "kv_heads", "head_dim", "rotary_dim", "axes", "interleaved", "pages", "page_size",
             "q", "k", "v", "q_out", "k_cache", "v_cache", "positions", "slots", "frequencies", "pair_axis")
    more = ("q_weight", "k_weight", "exponents", "eps", "bits8")
    a = dict(zip(names + more, [9, 3, 4, 2, 64, 64, 1, 0, 8, 16] + [4096] * 9 + [0] + [4096] * 3 + [1e-6, 1])) | change
    packed = paged._NORM_ROTATE_APPEND_ARGS.pack(*(a[n] for n in names), 256, 64, 128, 64, 128, 64, 256, 64, 2048, 128, 64, 2048, 128, 64, 3,
                                                 *(a[n] for n in more))
    assert native_lib.emmy_norm_rotate_append(packed, None) == -1
    said = native_lib.emmy_last_error()
    assert words in said and b"norm_rotate_append" in said, said


@pytest.mark.parametrize("q_lens", [[2], [100], [300]])
@pytest.mark.parametrize("change,words", [
    (dict(dtype=7), b"dtype"), (dict(scale=-1.0), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(scale=3.4e38), b"scale"),
    (dict(page_size=0), b"page_size"), (dict(page_size=24), b"page_size"), (dict(page_size=192), b"page_size"), (dict(pages=0), b"pages"), (dict(table_width=1), b"does not hold"), (dict(q=0), b"null"),
    (dict(scratch=0), b"null"), (dict(q=4104), b"16 bytes"), (dict(scratch=4112), b"16 bytes"), (dict(table=4098), b"16 bytes"),
    (dict(exponents=4098), b"16 bytes"), (dict(k_cache=4104), b"16 bytes"), (dict(q_token=100), b"stride"), (dict(k_page=-2048), b"stride"),
    (dict(v_token=136), b"stride"), (dict(v_token=0), b"stride"),
])
def test_c_attention_refuses(native_lib, q_lens, change, words):
    plan = paged.QuantisedPlan(q_lens, [5000], 8, 2, 64, device="cpu", ctas=148)
    assert plan.scratch.numel()
    names = ("dtype", "pages", "page_size", "table_width", "scale", "q", "out", "lse", "k_cache", "v_cache", "table",
             "plan_words", "scratch", "q_token", "q_head", "out_token", "out_head", "k_page", "k_token", "k_head",
             "v_page", "v_token", "v_head", "table_stride", "exponents")
    a = dict(zip(names, [9, 400, 16, 400, 0.125] + [4096] * 8 + [512, 64, 512, 64, 2048, 128, 64, 2048, 128, 64, 400, 4096])) | change
    assert native_lib.emmy_quantised_attention(plan._h, paged._QUANTISED_ATTENTION_ARGS.pack(*a.values()), None) == -1
    assert words in native_lib.emmy_last_error(), native_lib.emmy_last_error()


@pytest.mark.parametrize("change,words", [
    (dict(dtype=8), b"dtype"), (dict(sequences=-1), b"count"), (dict(rows=-1), b"count"), (dict(drafts=-1), b"count"), (dict(drafts=9), b"count"),
    (dict(vocabulary=0), b"vocabulary"), (dict(target=0), b"null"), (dict(drafted=0), b"null"), (dict(tokens=0), b"null"),
    (dict(target=4098), b"multiple"), (dict(first=4098), b"multiple"), (dict(target_stride=-5), b"stride"),
])
def test_c_verify_refuses(native_lib, change, words):
    names = ("dtype", "sequences", "rows", "drafts", "vocabulary", "reserved", "target", "proposal", "drafted", "uniforms", "finals", "first",
             "accepted", "tokens", "target_stride", "proposal_stride")
    a = dict(zip(names, [7, 2, 8, 6, 100, 0] + [4096] * 8 + [100, 100])) | change
    assert native_lib.emmy_verify(paged._VERIFY_ARGS.pack(*a.values()), None) == -1
    assert words in native_lib.emmy_last_error(), native_lib.emmy_last_error()
    assert native_lib.emmy_verify(paged._VERIFY_ARGS.pack(*(a | dict(zip(names, [7, 0, 0, 0, 5]))).values()), None) == 0
