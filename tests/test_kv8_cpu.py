"""The 8-bit paged KV cache and sm_draw without a device: arguments that the
entry points refuse before they touch a GPU, and the 64-bit statements the GPU
tests compare with (tests/kv8_ref.py) against each other and by hand."""
import ctypes as C

import numpy as np
import pytest

import kv8_ref as ref
import smotor

ARG = 1  # SM_ERR_ARG
OK = 0x1000  # an aligned non-null address; nothing reads it


def refused(call):
    with pytest.raises(smotor.EngineError) as e:
        call()
    assert e.value.status == ARG, str(e.value)


def plan(**kw):
    a = dict(n_seqs=2, lens=OK, add=OK, table=OK, table_ld=4, free=OK, n_free=OK, n_rows=2, lens_out=OK + 4096, first=OK,
             slots=OK, status=OK)
    a.update(kw)
    smotor.kv_plan(**a)


@pytest.mark.parametrize("kw", [
    dict(n_seqs=16385), dict(n_rows=1 << 31), dict(table_ld=1 << 31), dict(lens_out=OK), dict(lens=0), dict(add=0),
    dict(table=0), dict(n_free=0), dict(lens_out=0), dict(first=0), dict(slots=0), dict(status=0), dict(lens=OK + 2),
    dict(slots=OK + 4)])
def test_plan_refuses(kw):
    refused(lambda: plan(**kw))


def cache(**kw):
    a = dict(codes=OK, scales=OK, n_pages=4, n_kv_heads=2, head_dim=64, fmt=smotor.KV8_E4M3)
    a.update(kw)
    return smotor.Kv8Cache(**a)


@pytest.mark.parametrize("kw", [dict(fmt=2), dict(head_dim=0), dict(head_dim=24), dict(head_dim=144), dict(n_kv_heads=0),
                                dict(n_kv_heads=1025), dict(n_pages=0), dict(n_pages=1 << 31), dict(codes=0),
                                dict(codes=OK + 8)])
def test_cache_descriptions_refused(kw):
    refused(lambda: cache(**kw).append(OK, OK, smotor.F32, 1, OK))


@pytest.mark.parametrize("kw", [dict(dtype=smotor.Q8_0), dict(n_rows=1 << 31), dict(ld_k=64), dict(ld_v=130),
                                dict(ld_k=1 << 32)])
def test_append_refuses(kw):
    a = dict(k=OK, v=OK, dtype=smotor.F32, n_rows=1, slots=OK)
    a.update(kw)
    refused(lambda: cache().append(**a))


def test_append_of_no_rows_is_nothing():
    cache().append(0, 0, smotor.F32, 0, 0)


class OneWorkspace:
    h = C.create_string_buffer(64)  # read as device 0; the refusals come before


# sm_kv_plan reads its inputs again after other CTAs have written; sm_draw likewise
A = 1 << 20
PLAN = dict(n_seqs=40, lens=A, add=2 * A, table=3 * A, table_ld=4, free=4 * A, n_free=5 * A, n_rows=50, lens_out=6 * A,
            first=7 * A, slots=8 * A, pos=9 * A, seq=10 * A, status=11 * A)


@pytest.mark.parametrize("out,other", [
    ("lens_out", "lens"), ("lens_out", "add"), ("status", "n_free"), ("first", "add"), ("slots", "lens"), ("pos", "seq"),
    ("seq", "slots"), ("table", "lens"), ("table", "free"), ("status", "first"), ("lens_out", "first")])
@pytest.mark.parametrize("shift", [0, 8, -8])
def test_plan_refuses_outputs_over_other_arguments(out, other, shift):
    if shift == 8 and other in ("n_free", "free"):
        shift = 0  # one entry of them is looked at
    if shift == -8 and out == "status":
        shift = -4
    with pytest.raises(smotor.EngineError, match="overlaps") as e:
        smotor.kv_plan(**{**PLAN, out: PLAN[other] + shift})
    assert e.value.status == ARG


@pytest.mark.parametrize("shift", [160, -160])
def test_plan_takes_neighbours(shift):
    with pytest.raises(smotor.EngineError) as e:  # not the refusal: there is no such memory
        smotor.kv_plan(**{**PLAN, "lens_out": PLAN["lens"] + shift})
    assert "overlaps" not in str(e.value)


@pytest.mark.parametrize("kw,ok", [
    (dict(out=A), True), (dict(out=A, ld_q=1024, ld_out=512), False), (dict(out=A + 16), False), (dict(out=A - 512), False),
    (dict(out=A + 1024, ld_q=1024, ld_out=1024), True), (dict(out=A + 1024 + 2048, ld_q=1024, ld_out=1024), True),
    (dict(out=A - 1024, ld_q=1024, ld_out=1024), True), (dict(out=A + 4096 + 16, ld_q=1024, ld_out=1024), False),
    (dict(out=A + 1008, ld_q=1024, ld_out=1024), False), (dict(out=A + 9 * 1024), True)])
def test_attend_refuses_rows_that_overlap_otherwise(kw, ok):
    """9 f32 rows of 4 heads of 64: 1024 bytes each."""
    a = dict(q=A, dtype=smotor.F32, n_rows=9, n_heads=4, n_seqs=1, lens=4 * A, first=5 * A, table=6 * A, table_ld=1)
    with pytest.raises(smotor.EngineError) as e:  # where it takes them: there is no such memory
        cache().attend(OneWorkspace, **{**a, **kw})
    assert ("overlaps" in str(e.value)) == (not ok)


# A cache of 4 pages of 2 heads of 64: 32768 bytes of codes, 64 of scales. 9 f32 rows of K and V: 512 bytes each, of
# q and out (4 heads): 1024. CTAs read K, V, slots, lengths and tables after others have written.
@pytest.mark.parametrize("kw,ok", [
    (dict(), True), (dict(k=A + 32752), False), (dict(k=A + 32768), True), (dict(v=A - 16), False),
    (dict(v=A - 9 * 512), True), (dict(slots=2 * A), False), (dict(slots=2 * A - 64), False), (dict(slots=2 * A - 72), True),
    (dict(slots=A + 8), False), (dict(scales=A + 32760), False), (dict(k=A - 9 * 512, ld_k=1024), False), (dict(v=3 * A), True)])
def test_append_refuses_a_cache_over_other_arguments(kw, ok):
    a = dict(codes=A, scales=2 * A, k=3 * A, v=4 * A, slots=5 * A)
    a.update(kw)
    c = cache(codes=a.pop("codes"), scales=a.pop("scales"))
    with pytest.raises(smotor.EngineError) as e:  # where it takes them: there is no such memory
        c.append(dtype=smotor.F32, n_rows=9, **a)
    assert ("overlaps" in str(e.value)) == (not ok)


@pytest.mark.parametrize("kw,ok", [
    (dict(), True), (dict(out=A), False), (dict(out=A + 32768 - 16), False), (dict(out=A + 32768), True),
    (dict(out=2 * A + 48), False), (dict(lens=4 * A + 9 * 1024 - 4), False), (dict(lens=4 * A + 9 * 1024), True),
    (dict(lens=4 * A - 8), True), (dict(first=4 * A - 8), False), (dict(first=4 * A - 12), True),
    (dict(table=4 * A - 28), False), (dict(table=4 * A - 32), True), (dict(lens=6 * A, first=6 * A), True),
    (dict(lens=3 * A + 512), True), (dict(out=4 * A, ld_out=2048, lens=4 * A + 8 * 8192), False)])
def test_attend_refuses_out_over_other_arguments(kw, ok):
    a = dict(q=3 * A, out=4 * A, lens=5 * A, first=6 * A, table=7 * A, table_ld=4)
    with pytest.raises(smotor.EngineError) as e:
        cache(codes=A, scales=2 * A).attend(OneWorkspace, dtype=smotor.F32, n_rows=9, n_heads=4, n_seqs=2, **{**a, **kw})
    assert ("overlaps" in str(e.value)) == (not ok)


@pytest.mark.parametrize("kw", [dict(tokens=3 * A), dict(tokens=2 * A + 32), dict(tokens=A + 396), dict(logprobs=5 * A + 4),
                                dict(logprobs=4 * A - 4), dict(ld=1 << 32), dict(tokens=4 * A, ld=128, mask=4 * A - 1123)])
def test_draw_refuses_outputs_over_other_arguments(kw):
    a = dict(logits=A, dtype=smotor.F32, n_rows=9, vocab=100, params=2 * A, u=3 * A, tokens=5 * A, mask=4 * A)
    refused(lambda: smotor.draw(**{**a, **kw}))


class NoWorkspace:
    h = None


def test_attend_refuses_without_workspace():
    refused(lambda: cache().attend(NoWorkspace(), OK, OK, smotor.F32, 1, 4, 1, OK, OK, OK, 1))


def draw(**kw):
    a = dict(logits=OK, dtype=smotor.F32, n_rows=1, vocab=100, params=OK, u=OK, tokens=OK)
    a.update(kw)
    smotor.draw(**a)


@pytest.mark.parametrize("kw", [dict(dtype=smotor.Q6_K), dict(vocab=0), dict(vocab=524289), dict(ld=99),
                                dict(n_rows=65537), dict(logits=0), dict(logits=OK + 2)])
def test_draw_refuses(kw):
    refused(lambda: draw(**kw))


def test_draw_of_no_rows_is_nothing():
    draw(n_rows=0, logits=0, params=0, u=0, tokens=0)


def test_null_structs_and_outputs_refused():
    assert smotor.lib().sm_kv8_append(None, OK, OK, 0, 1, 0, 0, OK, None) == ARG
    assert smotor.lib().sm_kv8_ws_new(None) == ARG
    assert smotor.lib().sm_kv8_ws_free(None) == 0


# ------------------------------------------------- the statements themselves ----
def test_e4m3_against_torch():
    torch = pytest.importorskip("torch")
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).float().numpy().astype(np.float64)
    assert np.array_equal(ref.E4M3, want, equal_nan=True)
    r = np.random.default_rng(0)
    x = np.concatenate([r.normal(0, 100, 20000), r.normal(0, 0.01, 20000), ref.E4M3[:126] + np.diff(ref.E4M3[:127]) / 2,
                        [0.0, -0.0, 448.0, -448.0, 2.0**-10, 2.0**-11, 2.0**-12]])
    x = np.clip(x, -448, 448).astype(np.float32)
    got = ref.encode(x.astype(np.float64), "e4m3")
    assert np.array_equal(got, torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


@pytest.mark.parametrize("fmt", ["e4m3", "i8"])
def test_page_scale_is_the_smallest(fmt):
    r = np.random.default_rng(1)
    top = np.abs(r.normal(0, 1, 200)) * 2.0 ** r.integers(-80, 100, 200)
    top = np.concatenate([top, ref.TOP[fmt] * 2.0 ** r.integers(-60, 60, 20), [0.0]])
    s = ref.page_scale(top, fmt)
    assert np.all(top <= ref.TOP[fmt] * s) and np.all((top > ref.TOP[fmt] * s / 2) | (s == 2.0**-100))


def test_plan_by_hand():
    table = np.full((3, 3), -1)
    table[0, 0], table[2, 0] = 7, 8
    t, lens_out, first, slots, pos, seq, status = ref.plan([31, 0, 32], [2, 0, 1], table, [4, 5, 6], 3, 5)
    assert t[0, 1] == 6 and t[2, 1] == 5 and list(lens_out) == [33, 0, 33] and list(first) == [0, 2, 2, 3]
    assert list(slots) == [7 * 32 + 31, 6 * 32, 5 * 32, -1, -1] and list(pos) == [31, 32, 32, -1, -1]
    assert list(seq) == [0, 0, 2, -1, -1] and list(status) == [1, 0]


def test_draw_by_hand():
    x = np.log(np.array([1.0, 4.0, 2.0, 1.0]))
    assert [ref.draw(x, 1, 0, 1, 0, u)[0] for u in (0, 0.12, 0.13, 0.62, 0.63, 0.99)] == [0, 0, 1, 1, 2, 3]
    assert [ref.draw(x, 1, 2, 1, 0, u)[0] for u in (0, 0.66, 0.67)] == [1, 1, 2]
    assert [ref.draw(x, 1, 0, 0.5, 0, u)[0] for u in (0, 0.99)] == [1, 1]
    assert [ref.draw(x, 1, 0, 0.51, 0, u)[0] for u in (0, 0.99)] == [1, 2]
    assert [ref.draw(x, 1, 0, 1, 0.4, u)[0] for u in (0, 0.99)] == [1, 2]
    assert ref.draw(x, 0, 0, 1, 0, 0.5) == (1, 0.0) and ref.draw(x, 1, 0, 1, 0, 0.5, np.zeros(4))[0] == -1


def test_the_structs_have_the_headers_sizes():
    assert C.sizeof(smotor.sm_kv8) == 40 and C.sizeof(smotor.sm_draw_params) == 16
