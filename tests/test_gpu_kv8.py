"""The 8-bit paged KV cache's operators and sm_draw on the GPU, against their
plain statements in 64 bits (tests/kv8_ref.py).

Tolerances. plan: equal. append: equal (a code is the correctly rounded one).
attend, for a row of n positions, relative to M = sum p |v| / sum p (what
errors of weights scale with) and to the output itself:
- F32: q and w enter as hi + lo f16, within 2^-22 of the row's largest q and of
  w; a score t (log2 units) is then off by at most (2^-22 + D 2^-24) A + |t| 2^-23
  with A = scale log2e sum |q k|, and a weight by ln2 of that + 2^-22. The tests'
  A stays below 30 (|q k| averages 0.64 sigma_q sigma_k; sigma_k < 2.5 here), so a
  weight is within 2e-4 if all errors had one sign, and the output within that
  times M. Rounding errors have mixed signs: of D = 128 terms they grow as
  sqrt(D), which leaves 2e-5 M.
- F16, BF16: as above with q exact, w rounded to f16 (2^-11 of itself), the
  output rounded once (2^-11 f16, 2^-8 bf16 of the value).
draw: tokens equal; log probabilities to 2^-23 relative + 2e-7 (one rounding
to f32 of a value computed in f64 from weights off by 2^-44 each).
"""
import os
import subprocess
import sys

import numpy as np
import pytest

import kv8_ref as ref
import smotor

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

FMT = {"e4m3": smotor.KV8_E4M3, "i8": smotor.KV8_I8}
TYPES = {"f32": (torch.float32, smotor.F32), "f16": (torch.float16, smotor.F16), "bf16": (torch.bfloat16, smotor.BF16)}


def dev(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x))
    return (t if dtype is None else t.to(dtype)).cuda()


def stream():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------ plan ----
def run_plan(lens, add, table, free, n_free, n_rows, extras=True):
    n = len(lens)
    d = {k: dev(np.asarray(v, np.int32)) for k, v in dict(lens=lens, add=add, table=table, free=free, n_free=[n_free]).items()}
    i32 = dict(dtype=torch.int32, device="cuda")
    o = dict(lens_out=torch.full((n,), 99, **i32), first=torch.full((n + 1,), 99, **i32),
             slots=torch.full((n_rows,), 99, dtype=torch.int64, device="cuda"), pos=torch.full((n_rows,), 99, **i32),
             seq=torch.full((n_rows,), 99, **i32), status=torch.full((2,), 99, **i32))
    smotor.kv_plan(n, d["lens"].data_ptr(), d["add"].data_ptr(), d["table"].data_ptr(), d["table"].shape[1] if n else 0,
                   d["free"].data_ptr(), d["n_free"].data_ptr(), n_rows, o["lens_out"].data_ptr(), o["first"].data_ptr(),
                   o["slots"].data_ptr(), o["status"].data_ptr(), pos=o["pos"].data_ptr() if extras else 0,
                   seq=o["seq"].data_ptr() if extras else 0, stream=stream())
    return [d["table"].cpu().numpy()] + [o[k].cpu().numpy() for k in ("lens_out", "first", "slots", "pos", "seq", "status")]


def plan_case(n, most, new, rng, ld=None, short=None, pad=0):
    lens = rng.integers(0, most + 1, n)
    add = np.where(rng.random(n) < 0.3, rng.integers(0, new + 1, n), 1)
    ld = ld or (most + new + 31) // 32
    old = (lens + 31) // 32
    table = np.full((n, ld), -1)
    ids = rng.permutation(int(old.sum()) + 10 + int(((lens + add + 31) // 32 - old).sum()))
    at = 0
    for i in range(n):
        table[i, :min(ld, old[i])] = ids[at:at + old[i]][:ld]
        at += old[i]
    free = ids[at:]
    n_free = len(free) if short is None else min(short, len(free))
    return lens, add, table, free, n_free, max(0, int(add.sum()) + pad)


@pytest.mark.parametrize("n,most,new,short,pad", [
    (1, 0, 1, None, 0), (1, 64, 0, None, 3), (2, 33, 5, None, 0), (31, 200, 70, None, 5), (33, 40, 40, 4, 0),
    (100, 500, 100, 0, 1), (513, 100, 64, 300, 0), (1500, 300, 33, None, 700), (16384, 40, 2, None, 0), (300, 90, 40, None, -900)])
def test_plan(n, most, new, short, pad):
    c = plan_case(n, most, new, np.random.default_rng(n + most), short=short, pad=pad)
    for got, want in zip(run_plan(*c), ref.plan(*c)):
        assert np.array_equal(got, want)


def test_plan_full_rows_negative_lengths_and_bad_entries():
    lens = np.array([64, 63, -1, 5, 10, 2**31 - 1, 0])
    add = np.array([1, 1, 4, -7, 3, 2**31 - 1, 0])
    table = np.full((7, 2), -1)
    table[1] = [3, 4]  # sequence 3 and 4's tables hold no page: their slots are -1
    c = (lens, add, table, np.arange(10, 20), 10, 12)
    for got, want in zip(run_plan(*c), ref.plan(*c)):
        assert np.array_equal(got, want)


def test_plan_without_sequences_and_without_optional_outputs():
    got = run_plan([], [], np.zeros((0, 1)), [1], 1, 3)
    assert list(got[2]) == [0] and list(got[3]) == [-1] * 3 and list(got[6]) == [1, 0]
    c = plan_case(20, 100, 50, np.random.default_rng(3))
    got, want = run_plan(*c, extras=False), ref.plan(*c)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[3], want[3])


# ---------------------------------------------------------------- append ----
def pool(rng, P, H, D, fmt):
    codes = rng.integers(0, 256, (P, H, 2, 32, D)).astype(np.uint8)
    if fmt == "e4m3":
        codes[(codes & 127) == 127] = 0
    else:
        codes[codes == 128] = 0
    return codes, 2.0 ** rng.integers(-9, -2, (P, H, 2)).astype(np.float32)


def check_append(codes, scales, k, v, slots, fmt, ty, ld=0):
    dt, code = TYPES[ty]
    kd, vd = dev(k, dt), dev(v, dt)
    if ld:  # rows inside wider ones, as the parts of a fused projection
        wide = torch.full((k.shape[0], ld), float("nan"), dtype=dt, device="cuda")
        w = k.shape[1] * k.shape[2]
        wide[:, :w], wide[:, ld - w:] = kd.reshape(-1, w), vd.reshape(-1, w)
        kp, vp = wide.data_ptr(), wide[:, ld - w:].data_ptr()
    else:
        kp, vp = kd.data_ptr(), vd.data_ptr()
    cd, sd, sl = dev(codes), dev(scales), dev(np.asarray(slots, np.int64))
    c = smotor.Kv8Cache(cd.data_ptr(), sd.data_ptr(), codes.shape[0], codes.shape[1], codes.shape[4], FMT[fmt])
    c.append(kp, vp, code, len(slots), sl.data_ptr(), ld_k=ld, ld_v=ld, stream=stream())
    want_c, want_s = ref.append(codes, scales, kd.double().cpu().numpy(), vd.double().cpu().numpy(), slots, fmt)
    assert np.array_equal(sd.cpu().numpy(), want_s.astype(np.float32), equal_nan=True)
    assert np.array_equal(cd.cpu().numpy(), want_c)


def runs(rng, P, lengths, start=None):
    """Slots of sequences of the given row counts in pages of their own."""
    ids, out = list(rng.permutation(P)), []
    for n in lengths:
        off = int(rng.integers(0, 32)) if start is None else start
        page = ids.pop()
        for _ in range(n):
            out.append(page * 32 + off)
            off += 1
            if off == 32:
                off, page = 0, ids.pop()
    return out


@pytest.mark.parametrize("fmt", ["e4m3", "i8"])
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,D,lengths", [
    (1, 16, [1]), (2, 64, [1] * 9), (8, 128, [1] * 32), (2, 80, [32, 33, 1, 31]), (4, 128, [300]), (3, 112, [7, 64, 95, 2]),
    (1, 48, [2000])])
def test_append(fmt, ty, H, D, lengths):
    rng = np.random.default_rng(len(lengths) + D)
    P = sum(n // 32 + 3 for n in lengths)
    codes, scales = pool(rng, P, H, D, fmt)
    T = sum(lengths)
    mag = 2.0 ** rng.integers(-6, 5, (T, 1, 1))
    k, v = (rng.normal(0, 1, (T, H, D)) * mag for _ in range(2))
    check_append(codes, scales, k, v, runs(rng, P, lengths), fmt, ty)


@pytest.mark.parametrize("fmt", ["e4m3", "i8"])
def test_append_strided_rows_and_skipped_slots(fmt):
    rng = np.random.default_rng(5)
    codes, scales = pool(rng, 12, 2, 64, fmt)
    slots = runs(rng, 10, [40, 3])
    slots = [-1, -5] + slots + [12 * 32, 2**40, -1]
    k, v = (rng.normal(0, 1, (len(slots), 2, 64)) for _ in range(2))
    k[0], v[-1] = np.inf, np.nan  # of skipped rows
    check_append(codes, scales, k, v, slots, fmt, "bf16", ld=512)
    check_append(codes, scales, k, v, slots, fmt, "f32", ld=300)


@pytest.mark.parametrize("fmt", ["e4m3", "i8"])
def test_append_extremes(fmt):
    rng = np.random.default_rng(6)
    codes, scales = pool(rng, 9, 1, 16, fmt)
    top = ref.TOP[fmt]
    # zeros, the largest float, values next to a scale's border, tiny ones, ties between codes, NaN and infinity
    rows = np.zeros((8, 1, 16), np.float32)
    rows[1], rows[2, 0, 3] = np.finfo(np.float32).max, top
    rows[3, 0, 4] = np.nextafter(np.float32(top), np.float32(1e9))
    rows[4] = 1e-38
    rows[5, 0] = np.linspace(-top, top, 16).round() + 0.5
    rows[5, 0, 0], rows[6, 0, 1], rows[7, 0, 2] = top, np.nan, -np.inf
    check_append(codes, scales, rows, rows[::-1].copy(), [32 * i for i in range(8)], fmt, "f32")
    check_append(codes, scales, rows, rows, [32 * i + 5 for i in range(8)], fmt, "f32")
    scales[3] = np.nan  # a page spoilt earlier stays so until it begins anew
    check_append(codes, scales, rows[2:4], rows[2:4], [3 * 32 + 1, 3 * 32 + 2], fmt, "f32")
    check_append(codes, scales, rows[2:4], rows[2:4], [3 * 32, 3 * 32 + 1], fmt, "f32")


# ---------------------------------------------------------------- attend ----
def attend_state(rng, lens, rows, Hq, H, D, fmt, ty, ld=None, pad=0, spread=1.0):
    pages = [(max(l, 0) + 31) // 32 for l in lens]
    P = sum(pages) + 3
    ids = list(rng.permutation(P))
    table = np.full((len(lens), ld or max(1, max(pages, default=1))), -1, np.int32)
    for i, n in enumerate(pages):
        for j in range(min(n, table.shape[1])):
            table[i, j] = ids.pop()
    if fmt == "e4m3":
        codes = ref.encode(np.clip(rng.normal(0, 60, (P, H, 2, 32, D)), -448, 448), fmt)
    else:
        codes = np.clip(np.rint(rng.normal(0, 40, (P, H, 2, 32, D))), -127, 127).astype(np.int8).view(np.uint8)
    scales = (2.0 ** rng.integers(-8, -5, (P, H, 2))).astype(np.float32)
    scales[:, :, 1] *= (2.0 ** rng.integers(-3, 4, (P, H))).astype(np.float32)
    first = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    T = int(first[-1]) + pad
    q = rng.normal(0, spread, (T, Hq, D)).astype(np.float32)
    q = torch.from_numpy(q).to(TYPES[ty][0])
    return dict(codes=codes, scales=scales, table=table, first=first, lens=np.array(lens, np.int32), q=q, fmt=fmt, ty=ty)


def call_attend(s, ws=None, window=0, scale=None, ld=0, out=None, on=None):
    dt, code = TYPES[s["ty"]]
    P, H, _, _, D = s["codes"].shape
    T, Hq, _ = s["q"].shape
    d = {k: dev(s[k]) for k in ("codes", "scales", "table", "first", "lens")}
    w = Hq * D
    ld_ = ld or w
    q = torch.full((T, ld_), float("nan"), dtype=dt, device="cuda")
    q[:, :w] = s["q"].reshape(T, w).cuda()
    o = torch.full((T, ld_), 7.0, dtype=dt, device="cuda") if out is None else out
    c = smotor.Kv8Cache(d["codes"].data_ptr(), d["scales"].data_ptr(), P, H, D, FMT[s["fmt"]])
    ws = ws or smotor.Kv8Workspace()
    c.attend(ws, q.data_ptr(), o.data_ptr(), code, T, Hq, len(s["lens"]), d["lens"].data_ptr(), d["first"].data_ptr(),
             d["table"].data_ptr(), d["table"].shape[1], scale=scale, window=window, ld_q=ld, ld_out=ld, stream=stream())
    torch.cuda.synchronize()
    assert ld == 0 or bool((o[:, w:] == 7.0).all())
    return o[:, :w].reshape(T, Hq, D).double().cpu().numpy()


def check_attend(s, window=0, scale=None, **kw):
    got = call_attend(s, window=window, scale=scale, **kw)
    D = s["q"].shape[2]
    want, mag = ref.attend(s["codes"], s["scales"], s["fmt"], s["q"].double().numpy(), s["lens"], s["first"], s["table"],
                           D**-0.5 if scale is None else scale, window)
    rows = ~np.isnan(want).all((1, 2)) | (np.arange(len(want)) < s["first"][-1])
    assert np.all(got[~rows] == 7.0), "rows behind the last sequence were written"
    got, want, mag = got[rows], want[rows], mag[rows]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    eps = {"f32": 2e-5, "f16": 2.0**-11 + 2e-5, "bf16": 2.0**-11 + 2e-5}[s["ty"]]
    half = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}[s["ty"]]
    err = np.abs(got - want)[ok] - half * np.abs(want)[ok] - 2.0**-25
    assert err.size == 0 or np.all(err <= eps * mag[ok]), float((err / mag[ok]).max())


@pytest.mark.parametrize("fmt", ["e4m3", "i8"])
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("Hq,H,D", [(14, 2, 64), (8, 2, 128), (28, 4, 128), (4, 4, 80), (1, 1, 16), (24, 2, 96)])
def test_attend_single_tokens(fmt, ty, Hq, H, D):
    rng = np.random.default_rng(Hq + D)
    check_attend(attend_state(rng, [1, 2, 31, 32, 33, 100, 16, 17, 257], [1] * 9, Hq, H, D, fmt, ty))


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,lens,window", [
    ([5, 1, 0, 3], [70, 40, 12, 3], 0), ([40], [40], 0), ([17, 33], [200, 33], 0), ([5, 9], [90, 300], 20),
    ([3, 3], [100, 500], 1), ([70], [70], 33), ([2, 2], [64, 65], 1000)])
def test_attend_several_rows_and_windows(ty, rows, lens, window):
    rng = np.random.default_rng(sum(rows))
    check_attend(attend_state(rng, lens, rows, 14, 2, 64, "e4m3", ty, pad=3), window=window)
    check_attend(attend_state(rng, lens, rows, 4, 2, 128, "i8", ty), window=window)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_attend_long_sequences_share_ctas(ty):
    rng = np.random.default_rng(8)
    check_attend(attend_state(rng, [9000], [1], 7, 1, 128, "i8", ty))
    check_attend(attend_state(rng, [5000, 3, 0, 700, 1], [2, 1, 0, 1, 1], 8, 2, 64, "e4m3", ty))


@pytest.mark.parametrize("n", [300, 700])
def test_attend_many_short_sequences(n):
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 70, n)
    check_attend(attend_state(rng, list(lens), [1] * n, 4, 2, 64, "e4m3", "bf16"))
    check_attend(attend_state(rng, list(lens), list(np.minimum(lens, rng.integers(0, 3, n))), 2, 2, 32, "i8", "f32"))


# Many rows a sequence: the tensor-core form (256 rows on average, head_dim 64 or 128, 16-bit rows).
@pytest.mark.parametrize("fmt", ["e4m3", "i8"])
@pytest.mark.parametrize("ty", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,H,D", [(8, 2, 64), (14, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("rows,lens,window", [
    ([130, 1, 300], [200, 64, 300], 0), ([257], [257], 0), ([300, 290], [900, 290], 70), ([256], [5000], 0)])
def test_attend_many_rows(fmt, ty, Hq, H, D, rows, lens, window):
    if Hq == 4:
        rows, lens = [4 * r for r in rows], [max(4 * r, l) for r, l in zip(rows, lens)]
    rng = np.random.default_rng(sum(rows) + D)
    check_attend(attend_state(rng, lens, rows, Hq, H, D, fmt, ty, pad=2), window=window)


@pytest.mark.parametrize("D", [64, 128])
def test_attend_many_rows_at_the_edges(D):
    rng = np.random.default_rng(D)
    # more rows than positions, no rows, nothing held, a refused sequence
    s = attend_state(rng, [100, 50, 0, -1, 400], [300, 0, 20, 300, 400], 8, 2, D, "e4m3", "bf16", pad=5)
    check_attend(s)
    check_attend(s, scale=0.0)
    check_attend(s, scale=-0.3, ld=8 * D + 8)
    for i, n in enumerate(s["lens"]):  # codes behind the end
        if n > 0 and n % 32:
            s["codes"][s["table"][i, (n - 1) // 32], :, :, (n - 1) % 32 + 1:] = 0xFF
    check_attend(s)
    s["table"][4, 3], s["table"][4, 7], s["table"][0, 0] = -1, s["codes"].shape[0], 1 << 30
    check_attend(s)
    s["scales"][:, :, 1] *= (2.0 ** rng.integers(-40, 30, s["scales"].shape[:2])).astype(np.float32)
    s["scales"][:, :, 1] *= 1.37
    check_attend(s, window=90)


@pytest.mark.parametrize("ty,D", [("f16", 64), ("bf16", 128)])
def test_attend_many_rows_scales_of_any_fraction(ty, D):
    """Scales that are no powers of two, zeros and subnormals among V's: the same tolerance (an exponent off by
    2^-16 at most is 1.1e-5 of a weight)."""
    rng = np.random.default_rng(25)
    s = attend_state(rng, [1000, 700], [200, 260], 8, 2, D, "e4m3", ty)
    s["scales"] *= rng.uniform(1, 2, s["scales"].shape).astype(np.float32)
    check_attend(s)
    s["scales"][s["table"][0, 3], 0, 1], s["scales"][s["table"][1, 5], 1, 1] = 0.0, 1e-42
    check_attend(s, window=300)


def test_attend_many_rows_not_finite_scales():
    rng = np.random.default_rng(15)
    for which in (0, 1):
        s = attend_state(rng, [300], [300], 2, 1, 64, "e4m3", "f16")
        s["scales"][s["table"][0, 4], 0, which] = np.nan  # positions 128..159
        got = call_attend(s)
        assert np.isfinite(got[:128]).all() and np.isnan(got[128:]).all()
        got = call_attend(s, window=20)
        assert np.isnan(got[128:160]).all() and np.isfinite(got[179:]).all() and np.isfinite(got[:128]).all()


def test_attend_many_rows_repeat_bit_for_bit_and_status():
    rng = np.random.default_rng(16)
    s = attend_state(rng, [3000, 700], [300, 512], 14, 2, 64, "e4m3", "bf16")
    ws = smotor.Kv8Workspace()
    a = call_attend(s, ws=ws)
    for _ in range(3):
        assert np.array_equal(call_attend(s, ws=ws), a)
    ws.status(stream())


def test_attend_rows_that_see_nothing():
    rng = np.random.default_rng(9)
    s = attend_state(rng, [0, -1, 2, 40], [1, 2, 4, 1], 4, 2, 64, "e4m3", "f32", pad=2)  # row count above the length
    check_attend(s)
    s["table"][3] = -1  # no page of it in the pool
    check_attend(s)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_attend_bad_pages_take_no_part(ty):
    rng = np.random.default_rng(10)
    s = attend_state(rng, [200, 130, 500], [1, 2, 1], 4, 2, 64, "i8", ty, ld=10)  # the third is longer than its table
    s["table"][0, 2], s["table"][0, 5], s["table"][1, 0], s["table"][2, 1] = -1, 1 << 30, s["codes"].shape[0], -2**31
    check_attend(s)


@pytest.mark.parametrize("fmt", ["e4m3", "i8"])
@pytest.mark.parametrize("ty", ["f32", "f16"])
def test_attend_ignores_what_lies_behind_the_end(fmt, ty):
    """Codes behind a sequence's last position may be anything, E4M3's NaN among them."""
    rng = np.random.default_rng(11)
    s = attend_state(rng, [5, 33, 48], [1, 3, 1], 4, 2, 64, fmt, ty)
    for i, n in enumerate(s["lens"]):
        s["codes"][s["table"][i, (n - 1) // 32], :, :, (n - 1) % 32 + 1:] = 0x7F if i % 2 else 0xFF
    check_attend(s)


def test_attend_strides_scale_and_spread():
    rng = np.random.default_rng(12)
    s = attend_state(rng, [100, 64], [2, 1], 4, 2, 80, "e4m3", "bf16", pad=1)
    check_attend(s, ld=4 * 80 + 64)
    check_attend(s, scale=0.0)
    check_attend(s, scale=-0.3)
    s = attend_state(rng, [100, 64], [2, 1], 4, 2, 80, "e4m3", "f32", spread=1e-20)
    check_attend(s, scale=1e19)
    s = attend_state(rng, [300, 64], [1, 1], 4, 2, 64, "i8", "f32")
    s["scales"][:, :, 1] *= (2.0 ** rng.integers(-40, 30, s["scales"].shape[:2])).astype(np.float32)
    s["scales"][:, :, 1] *= 1.37  # not powers of two: a cache that another program wrote
    check_attend(s)


@pytest.mark.parametrize("ty,D,rows,length", [("f32", 64, 1, 300), ("f32", 128, 3, 9000), ("bf16", 128, 1, 9000),
                                              ("bf16", 64, 20, 300), ("bf16", 64, 300, 900), ("bf16", 128, 256, 2500)])
@pytest.mark.parametrize("low,high", [(-100, 66), (-60, 70), (-30, 90), (0, 118), (-20, 127)])
def test_attend_scales_of_v_of_any_spread(ty, D, rows, length, low, high):
    """A page of large values takes no part of the sum of weights away from pages whose scale is far smaller, in
    whatever order and in whatever parts they are met (zeros come with the smallest scale, 2^-100).
    Beside the tolerances above, weights x scale are f16 with the largest at 2^11 or more: a position is off by half
    a subnormal step, 2^-25, which is 2^-36 of the largest p s_v, times its code (at most 127). That is what an
    element is off by to which the largest page adds nothing."""
    rng = np.random.default_rng(length + high)
    pages = -(-length // 32)
    for at in ([0], [pages - 1], [pages // 2, 1]):
        s = attend_state(rng, [length, 33 + rows], [rows, rows], 4, 2, D, "i8", ty)
        s["q"] *= 0.25
        s["scales"][:, :, 1] = 2.0**low
        if low == -100:
            s["codes"][:, :, 1] = 0
            big = s["table"][0, at]
            s["codes"][big, :, 1] = rng.integers(-90, 91, s["codes"][big, :, 1].shape).astype(np.int8).view(np.uint8)
        if high == 127:  # the largest that f32 holds: 2^127 x 1
            s["codes"][:, :, 1] = np.clip(s["codes"][:, :, 1].view(np.int8), -1, 1).view(np.uint8)
        s["scales"][s["table"][0, at], :, 1] = 2.0**high
        got, q = call_attend(s), s["q"].double().numpy()
        want, mag = ref.attend(s["codes"], s["scales"], "i8", q, s["lens"], s["first"], s["table"], D**-0.5)
        flat = s["codes"].copy()  # V = 1 in the large pages, 0 elsewhere: their share of the sum is above their p
        flat[:, :, 1] = s["scales"][:, :, 1, None, None] == 2.0**high
        most = ref.attend(flat, s["scales"], "i8", q, s["lens"], s["first"], s["table"], D**-0.5)[0]
        half, eps = {"f32": (2.0**-24, 2e-5), "bf16": (2.0**-8, 2.0**-11 + 2e-5)}[ty]
        err = np.abs(got - want) - half * np.abs(want) - eps * mag - 2.0**-36 * 127 * length * most
        assert np.all(err <= 2.0**-126), (at, float(err.max()))


def test_attend_not_finite_scales_reach_the_rows_that_see_them():
    rng = np.random.default_rng(13)
    for which in (0, 1):
        s = attend_state(rng, [70, 70], [40, 1], 2, 1, 64, "e4m3", "f32")
        s["scales"][s["table"][0, 1], 0, which] = np.nan  # positions 32..63: rows from 32 on see them
        got = call_attend(s)
        assert np.isfinite(got[:2]).all() and np.isnan(got[2:40]).all() and np.isfinite(got[40]).all()


@pytest.mark.parametrize("ty,D,rows", [("f32", 64, 3), ("f16", 64, 3), ("bf16", 80, 9), ("f16", 64, 300), ("bf16", 128, 260)])
@pytest.mark.filterwarnings("ignore:invalid value")
def test_attend_rows_that_are_not_finite(ty, D, rows):
    """Of no use to others; NaN where they see something, however the signs fall, zeros where they do not."""
    rng = np.random.default_rng(28)
    s = attend_state(rng, [400, 2, 600], [rows, rows, 1], 4, 2, D, "i8", ty)
    s["codes"][:, :, 0, :, 5] = 100  # K's dim 5: all scores of a row with an infinity there have one sign
    for r, (h, d, x) in enumerate([(0, 5, np.inf), (1, 5, -np.inf), (2, 3, np.nan)]):
        for base in (0, 2 * rows - 3, rows):  # the last rows of the second sequence see its two positions, its first none
            s["q"][base + r, h, d] = float(x)
    check_attend(s)
    check_attend(s, window=1)


def test_attend_repeats_bit_for_bit_and_on_another_stream():
    rng = np.random.default_rng(14)
    s = attend_state(rng, [3000, 10, 900], [1, 1, 2], 14, 2, 64, "e4m3", "f32")
    ws = smotor.Kv8Workspace()
    a = call_attend(s, ws=ws)
    for _ in range(3):
        assert np.array_equal(call_attend(s, ws=ws), a)
    with torch.cuda.stream(torch.cuda.Stream()):
        assert np.array_equal(call_attend(s, ws=ws), a)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_attend_one_kv_head_for_many(ty):
    rng = np.random.default_rng(17)
    check_attend(attend_state(rng, [40, 100, 1], [1, 2, 1], 40, 1, 64, "e4m3", ty))


def test_attend_thousands_of_sequences():
    rng = np.random.default_rng(18)
    lens = rng.integers(0, 4, 5000)
    check_attend(attend_state(rng, list(lens), [1] * 5000, 1, 1, 16, "i8", "f32"))


@pytest.mark.parametrize("fmt,D", [("e4m3", 128), ("i8", 32)])
def test_attend_f32_keeps_its_bits_over_thousands_of_positions(fmt, D):
    """The 2-norm of the error: 6400 positions are 400 sums of 16, each rounded to 2^-24 of what is there: as a
    random walk 20 x 2^-24 = 1.2e-6; scores off by |t| 2^-23 ln2, |t| < 10, 0.8e-6; the rest is smaller. A sum
    cut off instead of rounded would be 400 x 2^-24 = 2.4e-5 low."""
    rng = np.random.default_rng(22)
    s = attend_state(rng, [6400, 6399], [40, 8], 4, 1, D, fmt, "f32")
    got = call_attend(s)
    want, _ = ref.attend(s["codes"], s["scales"], fmt, s["q"].double().numpy(), s["lens"], s["first"], s["table"], D**-0.5)
    assert np.linalg.norm(got - want) <= 4e-6 * np.linalg.norm(want)


@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("n,rows,D", [(300, 1, 128), (300, 1, 64), (150, 20, 128), (10, 400, 128), (10, 400, 64), (300, 1, 80)])
def test_attend_16_bit_rows_over_long_caches(n, rows, D, rising):
    """Sequences of 131072 positions, more than there are warps or CTAs to share one, over the same pages; V of one
    sign. The mean of the signed errors: outputs are rounded to nearest, weights (f16) too, so what is left is the
    tensor core's cut, 2^-23 of the sum a step of 16 positions, over the 128 steps (2048 positions) that it adds up by
    itself: 1.5e-5, and as much again for a sum that has just passed a power of two. Over all 8192 steps it would be
    up to 1e-3 (5.5e-4 was measured)."""
    rng = torch.Generator(device="cuda").manual_seed(27)
    H, L, dt = 8, 131072, torch.float16
    P = L // 32
    codes = torch.randint(0, 256, (P, H, 2, 32, D), generator=rng, dtype=torch.uint8, device="cuda")
    codes[codes == 128] = 0
    codes[:, :, 1] = torch.randint(64, 128, (P, H, 32, D), generator=rng, dtype=torch.uint8, device="cuda")
    scales = torch.full((P, H, 2), 2.0**-7, device="cuda")
    if rising:  # the largest contribution grows all the way
        scales[:, :, 1] = 2.0 ** (-13 + torch.arange(P, device="cuda") * 12 // P)[:, None]
    q = torch.randn((n * rows, H, D), generator=rng, device="cuda").to(dt)
    out = torch.zeros_like(q)
    i32 = dict(dtype=torch.int32, device="cuda")
    lens, first = torch.full((n,), L, **i32), torch.arange(n + 1, **i32) * rows
    table = torch.arange(P, **i32).repeat(n, 1)
    cache, ws = smotor.Kv8Cache(codes.data_ptr(), scales.data_ptr(), P, H, D, smotor.KV8_I8), smotor.Kv8Workspace()
    cache.attend(ws, q.data_ptr(), out.data_ptr(), smotor.F16, n * rows, H, n, lens.data_ptr(), first.data_ptr(),
                 table.data_ptr(), P, stream=stream())
    ws.status(stream())
    err = []
    picks = torch.arange(0, n * rows, max(1, n * rows // 40), device="cuda")  # rows looked at
    seen = L - rows + 1 + picks % rows
    for h in range(H):
        k = codes[:, h, 0].view(torch.int8).double().reshape(L, D) * 2.0**-7
        v = (codes[:, h, 1].view(torch.int8).double() * scales[:, h, 1, None, None].double()).reshape(L, D)
        t = q[picks, h].double() @ k.T * D**-0.5
        t[torch.arange(L, device="cuda")[None] >= seen[:, None]] = -torch.inf
        want = torch.softmax(t, 1) @ v
        got = out[picks, h].double()
        assert bool(((got - want).abs() <= (2.0**-11 + 2.0**-11 + 2e-5) * want).all())
        err.append(((got - want) / want).mean())
    assert abs(float(torch.stack(err).mean())) <= 3e-5


@pytest.mark.parametrize("ty,rows", [("f32", 3), ("bf16", 1), ("f16", 20), ("bf16", 300)])
@pytest.mark.parametrize("size", [1e9, 1e31])
def test_attend_of_huge_scores(ty, rows, size):
    """Scores so large that one position has all the weight, in steps of f32 wider than the exponents the weights
    are made of: the output is that position's V, rounded once."""
    if ty == "f16":
        size = 6e4 if size < 1e20 else 3e4
    rng = np.random.default_rng(23)
    s = attend_state(rng, [700, 90 + rows], [rows, rows], 4, 1, 64, "e4m3", ty)
    s["q"] = (s["q"].float() * size).clamp(-3e38, 3e38).to(s["q"].dtype) if ty != "f16" else (s["q"].float() * size / 8).to(s["q"].dtype)
    scale = 1e5 if ty == "f16" else 1.0
    q = s["q"].double().numpy()
    want, mag = ref.attend(s["codes"], s["scales"], "e4m3", q, s["lens"], s["first"], s["table"], scale)
    got = call_attend(s, scale=scale)
    assert np.all(np.isfinite(got))
    # rows whose two best scores differ by less than rounding moves them are left out: K is known, so look at it
    clear = leading(s, q) > 1e-5
    assert clear.mean() > 0.9
    half = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}[ty]
    err = np.abs(got - want) - half * np.abs(want) - (2.0**-11 + 2e-5 if ty != "f32" else 2e-5) * np.abs(mag)
    assert np.all(err[clear] <= 0)


def leading(s, q):
    """By how much each row's best score leads its second, relative to the largest one."""
    K = ref.E4M3[s["codes"][:, 0, 0].astype(int)] * s["scales"][:, 0, 0].astype(np.float64)[:, None, None]
    out = np.zeros(q.shape[:2])
    for i, n in enumerate(s["lens"]):
        r0, r1 = s["first"][i], s["first"][i + 1]
        k = K[s["table"][i, :-(-n // 32)]].reshape(-1, q.shape[2])
        for r in range(r0, r1):
            t = np.sort(q[r] @ k[: n - (r1 - r0) + (r - r0) + 1].T, 1)
            out[r] = (t[:, -1] - t[:, -2]) / np.abs(t).max(1) if t.shape[1] > 1 else 1.0
    return out


@pytest.mark.parametrize("ty,D,rows", [("f32", 16, 1), ("bf16", 128, 1), ("f16", 64, 7), ("bf16", 128, 400)])
def test_attend_in_place_and_into_columns_beside_q(ty, D, rows):
    rng = np.random.default_rng(24)
    s = attend_state(rng, [3000, 17 + rows], [rows, rows], 4, 2, D, "i8", ty)
    want = call_attend(s)
    d = {k: dev(s[k]) for k in ("codes", "scales", "table", "first", "lens")}
    cache, ws = smotor.Kv8Cache(d["codes"].data_ptr(), d["scales"].data_ptr(), len(s["codes"]), 2, D, smotor.KV8_I8), smotor.Kv8Workspace()
    both = torch.full((2 * rows, 2, 4, D), 5.0, dtype=TYPES[ty][0], device="cuda")
    both[:, 1] = s["q"].cuda()
    q = s["q"].cuda().contiguous()
    for x, y, ld in ((q.data_ptr(), q.data_ptr(), 0), (both[:, 1].data_ptr(), both.data_ptr(), 8 * D)):
        cache.attend(ws, x, y, TYPES[ty][1], 2 * rows, 4, 2, d["lens"].data_ptr(), d["first"].data_ptr(),
                     d["table"].data_ptr(), s["table"].shape[1], ld_q=ld, ld_out=ld, stream=stream())
    torch.cuda.synchronize()
    assert np.array_equal(q.double().cpu().numpy(), want) and np.array_equal(both[:, 0].double().cpu().numpy(), want)
    assert torch.equal(both[:, 1].cpu(), s["q"])


def test_first_calls_of_a_process_are_captured():
    code = """
import torch, smotor
P = lambda *s, dt=torch.int32: torch.zeros(s, dtype=dt, device="cuda")
ws = smotor.Kv8Workspace()
codes, scales, q = P(4, 1, 2, 32, 64, dt=torch.uint8), P(4, 1, 2, dt=torch.float32), P(300, 4, 64, dt=torch.bfloat16)
kv, out = q[:, :1].contiguous() + 1, q + 7
lens, add, table, free, n_free = P(1), P(1) + 40, P(1, 4) - 1, P(4) + torch.arange(4, device="cuda", dtype=torch.int32), P(1) + 4
lens_out, first, slots, status = P(1), P(2), P(300, dt=torch.int64), P(2)
logits, par, u, tok = P(1, 100000, dt=torch.float32), torch.tensor([[1.0, 0, 0.9, 0]], device="cuda"), P(1, dt=torch.float32), P(1)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    s = torch.cuda.current_stream().cuda_stream
    c = smotor.Kv8Cache(codes.data_ptr(), scales.data_ptr(), 4, 1, 64)
    smotor.kv_plan(1, lens.data_ptr(), add.data_ptr(), table.data_ptr(), 4, free.data_ptr(), n_free.data_ptr(), 300,
                   lens_out.data_ptr(), first.data_ptr(), slots.data_ptr(), status.data_ptr(), stream=s)
    c.append(kv.data_ptr(), kv.data_ptr(), smotor.BF16, 300, slots.data_ptr(), stream=s)
    for n in (300, 40):
        c.attend(ws, q.data_ptr(), out.data_ptr(), smotor.BF16, n, 4, 1, lens_out.data_ptr(), first.data_ptr(),
                 table.data_ptr(), 4, stream=s)
    smotor.draw(logits.data_ptr(), smotor.F32, 1, 100000, par.data_ptr(), u.data_ptr(), tok.data_ptr(), stream=s)
g.replay()
torch.cuda.synchronize()
assert bool((out[:40] == 1).all()) and bool((out[40:] == 7).all()) and int(tok[0]) == 0 and int(status[0]) == 2
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, cwd=os.path.dirname(smotor.__path__[0]))


def test_attend_two_calls_at_once():
    rng = np.random.default_rng(19)
    states = [attend_state(rng, [6000, 200], [1, 1], 14, 2, 64, "e4m3", "f32"),
              attend_state(rng, [900, 700], [300, 300], 8, 2, 128, "i8", "bf16")]
    d, want, q, out, cache, ws = [], [], [], [], [], []
    for s in states:
        want.append(call_attend(s))
        d.append({k: dev(s[k]) for k in ("codes", "scales", "table", "first", "lens")})
        q.append(s["q"].cuda().contiguous())
        out.append(torch.zeros_like(q[-1]))
        P, H, _, _, D = s["codes"].shape
        cache.append(smotor.Kv8Cache(d[-1]["codes"].data_ptr(), d[-1]["scales"].data_ptr(), P, H, D, FMT[s["fmt"]]))
        ws.append(smotor.Kv8Workspace())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for i, s in enumerate(states):
            T, Hq, _ = s["q"].shape
            cache[i].attend(ws[i], q[i].data_ptr(), out[i].data_ptr(), TYPES[s["ty"]][1], T, Hq, 2, d[i]["lens"].data_ptr(),
                            d[i]["first"].data_ptr(), d[i]["table"].data_ptr(), s["table"].shape[1],
                            stream=streams[i].cuda_stream)
    torch.cuda.synchronize()
    for i in range(2):
        assert np.array_equal(out[i].double().cpu().numpy(), want[i])


@pytest.mark.parametrize("many", [False, True])
def test_pages_behind_four_gigabytes(many):
    """The same rows through low and through high pages of a pool of 4.5 GB."""
    rng = np.random.default_rng(20)
    P, D, n = 560000, 128, 300
    codes = torch.empty((P, 1, 2, 32, D), dtype=torch.uint8, device="cuda")
    scales = torch.ones((P, 1, 2), device="cuda")
    cache = smotor.Kv8Cache(codes.data_ptr(), scales.data_ptr(), P, 1, D)
    k, v = (dev(rng.normal(0, 1, (n, 1, D)), torch.bfloat16) for _ in range(2))
    rows = n if many else 1
    q = dev(rng.normal(0, 1, (rows, 2, D)), torch.bfloat16)
    lens, first = dev(np.array([n], np.int32)), dev(np.array([0, rows], np.int32))
    ws, got = smotor.Kv8Workspace(), []
    for base in (0, P - 10):
        pages = np.arange(base, base + 10)
        slots = dev((pages[np.arange(n) // 32] * 32 + np.arange(n) % 32).astype(np.int64))
        table, out = dev(pages.astype(np.int32)), torch.zeros_like(q)
        cache.append(k.data_ptr(), v.data_ptr(), smotor.BF16, n, slots.data_ptr(), stream=stream())
        cache.attend(ws, q.data_ptr(), out.data_ptr(), smotor.BF16, rows, 2, 1, lens.data_ptr(), first.data_ptr(),
                     table.data_ptr(), 10, stream=stream())
        torch.cuda.synchronize()
        got.append((codes[base:base + 10].cpu(), scales[base:base + 10].cpu(), out.float().cpu()))
    used = np.arange(320).reshape(10, 32) < n
    for a, b in zip(got[0], got[1]):
        if a.dtype == torch.uint8:
            a, b = (x[:, 0].transpose(1, 2)[torch.from_numpy(used)] for x in (a, b))
        assert torch.equal(a, b)
    assert bool(torch.isfinite(got[0][2]).all()) and float(got[0][2].abs().max()) > 0


def test_device_refusals():
    host = torch.zeros(4096, pin_memory=True)
    on = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda").data_ptr()
    c = smotor.Kv8Cache(on, on, 1, 1, 64)
    ws = smotor.Kv8Workspace()
    for call in (lambda: c.append(host.data_ptr(), on, smotor.F32, 1, on),
                 lambda: c.append(on, on, smotor.F32, 1, host.data_ptr()),
                 lambda: c.attend(ws, on, host.data_ptr(), smotor.F32, 1, 1, 1, on, on, on, 1),
                 lambda: c.attend(ws, on, on, smotor.F32, 1, 3, 1, on, on, on, 1, scale=float("nan")),
                 lambda: smotor.draw(on, smotor.F32, 1, 8, on, host.data_ptr(), on),
                 lambda: smotor.draw(np.zeros(8).ctypes.data, smotor.F32, 1, 8, on, on, on)):
        with pytest.raises(smotor.EngineError) as e:
            call()
        assert e.value.status == 1


# ------------------------------------------------------------------ draw ----
def check_draw(x, params, u, ty="f32", mask=None, ld=0):
    dt, code = TYPES[ty]
    n, V = x.shape
    xd = dev(x, dt)
    if ld:
        wide = torch.full((n, ld), 50.0, dtype=dt, device="cuda")
        wide[:, :V] = xd
        if mask is not None:
            mask = np.concatenate([mask, np.ones((n, ld - V), np.uint8)], 1)
    par = np.zeros(n, dtype=[("t", "f4"), ("k", "i4"), ("p", "f4"), ("m", "f4")])
    for i, q in enumerate(params):
        par[i] = q
    pd, ud = dev(par.view(np.uint8)), dev(np.asarray(u, np.float32))
    md = dev(mask) if mask is not None else None
    tok, lp = torch.full((n,), 77, dtype=torch.int32, device="cuda"), torch.full((n,), 77.0, device="cuda")
    smotor.draw((wide if ld else xd).data_ptr(), code, n, V, pd.data_ptr(), ud.data_ptr(), tok.data_ptr(),
                logprobs=lp.data_ptr(), mask=0 if md is None else md.data_ptr(), ld=ld, stream=stream())
    tok, lp, xs = tok.cpu().numpy(), lp.cpu().numpy(), xd.double().cpu().numpy()
    for i in range(n):
        t, l = ref.draw(xs[i], *[float(par[i][f]) if f != "k" else int(par[i][f]) for f in ("t", "k", "p", "m")], u[i],
                        None if mask is None else mask[i, :V])
        assert tok[i] == t, (i, params[i], u[i], tok[i], t)
        assert lp[i] == l or abs(lp[i] - l) <= 2.0**-23 * abs(l) + 2e-7, (i, params[i], lp[i], l)


PARAMS = [(1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.0, 40, 0.9, 0.0), (1.3, 0, 0.95, 0.0), (1.0, 0, 1.0, 0.05),
          (0.9, 60, 0.8, 0.02), (0.0, 5, 0.5, 0.5), (-1.0, 0, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0),
          (1.0, 0, 1.0, 2.0), (1e-3, 0, 0.9, 0.0), (100.0, 0, 0.5, 0.0), (1.0, 1500, 0.99, 0.0), (2.0, 0, 0.3, 1e-3),
          (1.0, 10**9, 2.0, -1.0), (1e-42, 0, 0.9, 0.0), (float("inf"), 0, 0.5, 0.0), (float("nan"), 0, 0.5, 0.0)]


@pytest.mark.parametrize("V", [1, 2, 7, 100, 1023, 4097, 32000, 152064])
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
def test_draw(V, ty):
    rng = np.random.default_rng(V)
    x = rng.normal(0, 2.5, (len(PARAMS), V))
    check_draw(x, PARAMS, rng.random(len(PARAMS)).astype(np.float32), ty)


@pytest.mark.parametrize("kind", ["flat", "tied", "peaked", "wide", "masked"])
def test_draw_distributions(kind):
    rng = np.random.default_rng(3)
    V, n = 50000, 24
    x = {"flat": np.zeros((n, V)), "tied": np.round(rng.normal(0, 2, (n, V)) * 2) / 2,
         "peaked": np.where(np.arange(V) == 777, 40.0, rng.normal(0, 1, (n, V))), "wide": rng.normal(0, 300, (n, V)),
         "masked": np.where(rng.random((n, V)) < 0.99, -np.inf, rng.normal(0, 1, (n, V)))}[kind].astype(np.float32)
    params = [(1.0, 0, 0.51, 0.0), (1.0, 3000, 1.0, 0.0), (1.0, 3001, 0.71, 0.0), (0.8, 0, 1.0, 0.1), (1.0, 49999, 0.999, 0.0),
              (5.0, 50, 0.93, 0.0)] * 4
    check_draw(x, params, rng.random(n).astype(np.float32), ld=50008)


def test_draw_edges():
    V = 300
    x = np.zeros((10, V), np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 5], x[2, 9] = np.inf, np.inf
    x[3, ::2] = np.nan
    x[4], x[4, 299] = -np.finfo(np.float32).max, -np.finfo(np.float32).max
    x[5] = np.linspace(-1e38, 1e38, V)
    x[6, :] = -0.0
    x[6, 3] = 0.0
    mask = np.ones((10, V), np.uint8)
    mask[7] = 0
    mask[8, :-1] = 0
    u = np.array([0.5, 0.5, 0.7, 0.0, 0.999, 0.3, 0.0, 0.5, 0.9, 0.25], np.float32)
    for p in [(1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 3, 0.7, 0.0), (1.0, 0, 0.51, 0.1)]:
        check_draw(x, [p] * 10, u, mask=mask)
    # numbers outside [0, 1) count as its ends
    check_draw(np.zeros((4, V)), [(1.0, 0, 1.0, 0.0)] * 4, np.array([1.0, -3.0, np.inf, np.nan], np.float32))


@pytest.mark.parametrize("V", [300, 1000, 50000])
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
def test_draw_values_whose_distance_overflows(V, ty):
    """Ordinary logits among some so far below the maximum that the distance in units of the temperature is no
    finite f32, below the 1024 values that are ordered at once; an earlier draw left larger values everywhere."""
    rng = np.random.default_rng(V + len(ty))
    check_draw(rng.normal(30, 3, (40, 60000)), [(1.0, 500, 0.9, 0.0)] * 40, rng.random(40).astype(np.float32), ty)
    params = [(1.0, k, p, 0.0) for k in (0, 20, 110, 200, 290, 590, 999) for p in (1.0, 0.9, 0.9999, 1 - 2.0**-23) if k or p < 1]
    params += [(1e-37, 0, 0.9, 0.0), (1e-37, 250, 0.9, 0.0), (1e-37, 0, 1 - 2.0**-23, 0.1), (1e38, 0, 0.6, 0.0),
               (1e38, 250, 1.0, 0.0), (float("inf"), 0, 0.7, 0.0), (float("inf"), 200, 0.99, 0.0)]
    n, info = len(params), torch.finfo(TYPES[ty][0])
    x = rng.normal(0, 2, (n, V))
    x[np.arange(n), rng.integers(0, V, n)] = 12.0  # peaked
    x = np.where(rng.random((n, V)) < 0.6, rng.choice([info.min, info.min / 2, -1e37 if ty != "f16" else -6e4], (n, V)), x)
    x[::3, 7] = np.inf
    x[1::3, 9] = info.max / 8
    mask = None
    if V > 1000:
        mask = (rng.random((n, V)) < 600 / V).astype(np.uint8)
    check_draw(x.astype(np.float32), params, rng.random(n).astype(np.float32), ty, mask=mask)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_draw_tiny_temperatures(ty):
    """Logits of the temperature's size down to the smallest floats, zeros and subnormal ones among them."""
    rng = np.random.default_rng(29)
    temps = [1e-20, 1e-26, 3e-30, 1e-36, 1e-37, 3e-38, 1e-38, 1e-39]
    params = [(t, k, p, m) for t in temps for k, p, m in [(0, 1.0, 0.0), (40, 0.9, 0.0), (0, 0.7, 0.0), (0, 1.0, 0.2)]]
    for shift in (0.0, -2.0, 3.0, 1e12):
        t = np.array([q[0] for q in params])[:, None]
        x = (rng.normal(0, 1.5, (len(params), 500)) + shift) * t
        x[:, ::7] = 0.0 if shift < 1e12 else x[:, ::7]
        check_draw(x.astype(np.float32), params, rng.random(len(params)).astype(np.float32), ty)


def test_draw_largest_vocabulary():
    rng = np.random.default_rng(4)
    check_draw(rng.normal(0, 1, (6, 524288)).astype(np.float32), PARAMS[:6], rng.random(6).astype(np.float32))


def test_draw_frequencies():
    """Equally spaced numbers draw each token as often as its probability says, within one."""
    n = 4096
    w = np.array([5.0, 1.0, 0.0, 3.0, 7.0])
    with np.errstate(divide="ignore"):
        x = np.tile(np.log(w).astype(np.float32), (n, 1))
    xd = dev(x)
    par = np.zeros(n, dtype=[("t", "f4"), ("k", "i4"), ("p", "f4"), ("m", "f4")])
    par[:] = (1.0, 0, 1.0, 0.0)
    pd, ud = dev(par.view(np.uint8)), dev((np.arange(n) / n).astype(np.float32))
    tok = torch.zeros(n, dtype=torch.int32, device="cuda")
    smotor.draw(xd.data_ptr(), smotor.F32, n, 5, pd.data_ptr(), ud.data_ptr(), tok.data_ptr())
    got = np.bincount(tok.cpu().numpy(), minlength=5)
    assert np.all(np.abs(got - n * w / w.sum()) <= 1)


# ------------------------------------------------------- the step together ----
@pytest.mark.parametrize("fmt,ty", [("e4m3", "bf16"), ("i8", "f32")])
@pytest.mark.parametrize("graph", [False, True])
def test_serving_steps(fmt, ty, graph):
    """Prompts, then decoding steps of a padded batch: plan -> append -> attend
    -> draw, eagerly or as one captured graph replayed each step; every step
    against the plain statements of the same operators."""
    rng = np.random.default_rng(21)
    dt, code = TYPES[ty]
    n, H, Hq, D, V, P, ld = 5, 2, 8, 64, 1000, 40, 8
    i32 = dict(dtype=torch.int32, device="cuda")
    codes, scales = torch.zeros((P, H, 2, 32, D), dtype=torch.uint8, device="cuda"), torch.zeros((P, H, 2), device="cuda")
    codes.fill_(0x7F)  # a fresh pool holds anything
    table = torch.full((n, ld), -1, **i32)
    free, n_free = torch.arange(P - 1, -1, -1, **i32), torch.tensor([P], **i32)
    lens, lens_out = torch.zeros(n, **i32), torch.zeros(n, **i32)
    adds = [np.array([33, 64, 1, 0, 90])] + [np.array([1, 1, 1, 0, 1])] * 3 + [np.array([1, 1, 1, 20, 1])]
    T = 200
    add, first, slots = torch.zeros(n, **i32), torch.zeros(n + 1, **i32), torch.zeros(T, dtype=torch.int64, device="cuda")
    status, pos, seq = torch.zeros(2, **i32), torch.zeros(T, **i32), torch.zeros(T, **i32)
    k, v, q = (torch.zeros((T, h, D), dtype=dt, device="cuda") for h in (H, H, Hq))
    out = torch.zeros((T, Hq, D), dtype=dt, device="cuda")
    logits, u = torch.zeros((n, V), device="cuda"), torch.zeros(n, device="cuda")
    par = np.zeros(n, dtype=[("t", "f4"), ("k", "i4"), ("p", "f4"), ("m", "f4")])
    par[:] = (1.0, 40, 0.9, 0.01)
    params, tok = dev(par.view(np.uint8)), torch.zeros(n, **i32)
    cache, ws = smotor.Kv8Cache(codes.data_ptr(), scales.data_ptr(), P, H, D, FMT[fmt]), smotor.Kv8Workspace()

    def step():
        st = stream()
        smotor.kv_plan(n, lens.data_ptr(), add.data_ptr(), table.data_ptr(), ld, free.data_ptr(), n_free.data_ptr(), T,
                       lens_out.data_ptr(), first.data_ptr(), slots.data_ptr(), status.data_ptr(), pos=pos.data_ptr(),
                       seq=seq.data_ptr(), stream=st)
        cache.append(k.data_ptr(), v.data_ptr(), code, T, slots.data_ptr(), stream=st)
        cache.attend(ws, q.data_ptr(), out.data_ptr(), code, T, Hq, n, lens_out.data_ptr(), first.data_ptr(),
                     table.data_ptr(), ld, stream=st)
        smotor.draw(logits.data_ptr(), smotor.F32, n, V, params.data_ptr(), u.data_ptr(), tok.data_ptr(), stream=st)

    g = None
    if graph:
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            step()
    for a in adds:
        add.copy_(dev(a.astype(np.int32)))
        for x in (k, v, q):
            x.copy_(dev(rng.normal(0, 1, x.shape).astype(np.float32)))
        logits.copy_(dev(rng.normal(0, 2, (n, V)).astype(np.float32)))
        u.copy_(dev(rng.random(n).astype(np.float32)))
        out.fill_(7.0)
        h = {m: x.cpu().numpy() for m, x in dict(lens=lens, table=table, free=free, codes=codes, scales=scales).items()}
        held = int(n_free.cpu()[0])
        (g.replay if g else step)()
        torch.cuda.synchronize()
        want = ref.plan(h["lens"], a, h["table"], h["free"], held, T)
        for got, w in zip((table, lens_out, first, slots, pos, seq, status), want):
            assert np.array_equal(got.cpu().numpy(), w)
        cw, sw = ref.append(h["codes"], h["scales"], k.double().cpu().numpy(), v.double().cpu().numpy(), want[3], fmt)
        assert np.array_equal(codes.cpu().numpy(), cw) and np.array_equal(scales.cpu().numpy(), sw.astype(np.float32))
        ow, mag = ref.attend(cw, sw, fmt, q.double().cpu().numpy(), want[1], want[2], want[0], D**-0.5)
        got = out.double().cpu().numpy()
        R = int(want[2][-1])
        assert np.all(got[R:] == 7.0)
        half = {"f32": 2.0**-24, "bf16": 2.0**-8}[ty]
        eps = {"f32": 2e-5, "bf16": 2.0**-11 + 2e-5}[ty]
        assert np.all(np.abs(got[:R] - ow[:R]) <= half * np.abs(ow[:R]) + eps * mag[:R])
        lg = logits.double().cpu().numpy()
        for i in range(n):
            assert int(tok[i]) == ref.draw(lg[i], 1.0, 40, float(np.float32(0.9)), float(np.float32(0.01)), float(u[i]))[0]
        lens.copy_(lens_out)
        n_free.copy_(status[:1])


@pytest.mark.parametrize("graph", [False, True])
def test_serving_when_the_pool_runs_short(graph):
    """A sequence that gets no pages keeps its length and its pages, and goes on when another one's are free."""
    rng = np.random.default_rng(26)
    n, H, Hq, D, P, ld, T = 3, 1, 2, 64, 6, 4, 120
    i32 = dict(dtype=torch.int32, device="cuda")
    codes, scales = torch.full((P, H, 2, 32, D), 0x7F, dtype=torch.uint8, device="cuda"), torch.zeros((P, H, 2), device="cuda")
    table, free, n_free = torch.full((n, ld), -1, **i32), torch.arange(P, **i32), torch.tensor([P], **i32)
    lens, lens_out, add, first = (torch.zeros(m, **i32) for m in (n, n, n, n + 1))
    slots, status = torch.zeros(T, dtype=torch.int64, device="cuda"), torch.zeros(2, **i32)
    k, v, q = (torch.zeros((T, h, D), device="cuda") for h in (H, H, Hq))
    out = torch.zeros((T, Hq, D), device="cuda")
    cache, ws = smotor.Kv8Cache(codes.data_ptr(), scales.data_ptr(), P, H, D), smotor.Kv8Workspace()

    def step():
        smotor.kv_plan(n, lens.data_ptr(), add.data_ptr(), table.data_ptr(), ld, free.data_ptr(), n_free.data_ptr(), T,
                       lens_out.data_ptr(), first.data_ptr(), slots.data_ptr(), status.data_ptr(), stream=stream())
        cache.append(k.data_ptr(), v.data_ptr(), smotor.F32, T, slots.data_ptr(), stream=stream())
        cache.attend(ws, q.data_ptr(), out.data_ptr(), smotor.F32, T, Hq, n, lens_out.data_ptr(), first.data_ptr(),
                     table.data_ptr(), ld, stream=stream())
        lens.copy_(torch.where(lens_out >= 0, lens_out, lens))
        n_free.copy_(status[:1])

    g = None
    if graph:
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            step()
    held = []
    for a in ([40, 33, 20], [30, 40, 1], [0, 40, 1], [0, 40, 1], [33, 1, 1]):
        if len(held) == 3:  # the first sequence has ended
            f, at = free.cpu().numpy(), int(n_free[0])
            f[at:at + 3] = table[0, :3].cpu().numpy()
            free.copy_(dev(f))
            n_free += 3
            lens[0] = 0
        add.copy_(dev(np.array(a, np.int32)))
        for x in (k, v, q):
            x.copy_(dev(rng.normal(0, 1, x.shape).astype(np.float32)))
        h = {m: x.cpu().numpy() for m, x in dict(lens=lens, table=table, free=free, codes=codes, scales=scales).items()}
        want = ref.plan(h["lens"], a, h["table"], h["free"], int(n_free[0]), T)
        (g.replay if g else step)()
        torch.cuda.synchronize()
        cw, sw = ref.append(h["codes"], h["scales"], k.double().cpu().numpy(), v.double().cpu().numpy(), want[3], "e4m3")
        assert np.array_equal(codes.cpu().numpy(), cw) and np.array_equal(table.cpu().numpy(), want[0])
        ow, mag = ref.attend(cw, sw, "e4m3", q.double().cpu().numpy(), want[1], want[2], want[0], D**-0.5)
        R = int(want[2][-1])
        assert np.all(np.abs(out.double().cpu().numpy()[:R] - ow[:R]) <= 2.0**-24 * np.abs(ow[:R]) + 2e-5 * mag[:R])
        held.append(lens.tolist())
    assert held == [[40, 33, 20], [70, 33, 21], [70, 33, 22], [0, 73, 23], [33, 74, 24]]
