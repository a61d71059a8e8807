"""Logit adjustment (fsb_adjust_logits) against a plain implementation in 64 bits: types, strides, offsets, windows, biases,
masks that leave a row empty, and what lies where a mask forbids.

Tolerance, before the output's own rounding: every step is one fp32 operation (relative error 2^-24 of its result), tanhf is within
2 ulp of a value below 1 (2^-22 with its argument's rounding), so |error| <= 2^-24 * 6 * (|x| + |f c| + |q| + |b|) + cap * 2^-21, with |x|
after the repetition penalty; the output's rounding adds half a step, eps / 2 relative (fp16: at least 2^-25, half its smallest step)."""
import numpy as np
import pytest

import ferro_b200 as fb

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16} if hasattr(torch, "float32") else {}
INF = float("inf")


def plain(logits, V, hists, rep, freq, pres, bias, allowed, cap, offset=0):
    """float64 result and the magnitudes that the tolerance counts"""
    x = logits[:, :V].double().cpu().numpy()
    out, mag = np.empty_like(x), np.empty_like(x)
    with np.errstate(invalid="ignore"):
        for r in range(x.shape[0]):
            y = x[r].copy()
            if cap:
                y = cap * np.tanh(y / cap)
            m = np.abs(y)
            ids = np.asarray(hists[r], dtype=np.int64) - offset
            ids, c = np.unique(ids[(ids >= 0) & (ids < V)], return_counts=True)
            z = y[ids]
            z = np.where(z > 0, z / np.float64(np.float32(rep[r])), z * np.float64(np.float32(rep[r])))
            f, q = np.float64(np.float32(freq[r])), np.float64(np.float32(pres[r]))
            m[ids] = np.maximum(np.abs(z), m[ids]) + np.abs(f) * c + np.abs(q)
            y[ids] = z - f * c - q
            for i, b in bias[r].items():
                if 0 <= i - offset < V:
                    y[i - offset] = -INF if b == -INF else y[i - offset] + np.float64(np.float32(b))
                    m[i - offset] += 0 if b == -INF else abs(b)
            if allowed[r] is not None:
                y[~allowed[r]] = -INF
            out[r], mag[r] = y, m
    return out, mag


def check(got, want, mag, cap, out_type):
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    big = {"f32": 3.4e38, "bf16": 3.38e38, "f16": 65504.0}[out_type]
    fits = ~inf & ~np.isnan(want) & (np.abs(want) < big)
    assert np.array_equal(got[inf], want[inf])
    half = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[out_type]
    tol = 2.0 ** -24 * 6 * mag[fits] + (cap * 2.0 ** -21 if cap else 0.0)
    tol = tol + half * (np.abs(want[fits]) + tol) + (2.0 ** -25 if out_type == "f16" else 0.0)
    worst = np.abs(got[fits] - want[fits]) - tol
    assert worst.size == 0 or worst.max() <= 0, (worst.max(), np.unravel_index(np.argmax(worst), worst.shape))


def pack(allowed, words, offset=0):
    """[rows][V] truth values as mask words (a device tensor); bits before the offset and behind the row are set at random"""
    rng = np.random.default_rng(5)
    bits = rng.random((len(allowed), words * 32)) < 0.5
    for r, a in enumerate(allowed):
        bits[r, offset:offset + len(a)] = a
    w = (bits.reshape(len(allowed), words, 32).astype(np.uint64) << np.arange(32, dtype=np.uint64)).sum(axis=2)
    return torch.from_numpy(w.astype(np.uint32).view(np.int32)).cuda()


def settings(rng, rows, V, hist, n_bias, offset=0, last_n=-1):
    rep = rng.choice([1.0, 1.1, 1.7, 0.6], rows).astype(np.float32)
    freq = rng.choice([0.0, 0.5, -0.25, 1.3], rows).astype(np.float32)
    pres = rng.choice([0.0, 0.75, -0.4], rows).astype(np.float32)
    hists = [rng.integers(offset - 3, offset + V + 3, int(rng.integers(0, hist + 1))).astype(np.int32) for _ in range(rows)]
    for h in hists:      # some tokens again and again
        if len(h) > 4:
            h[: len(h) // 2] = rng.choice(h[:3], len(h) // 2)
    bias = []
    for r in range(rows):
        ids = rng.permutation(np.arange(offset - 1, offset + V + 1))[: int(rng.integers(0, n_bias + 1))]
        bias.append({int(i): float(np.float32(v)) for i, v in zip(ids, rng.choice([-100.0, -1.5, 0.0, 2.25, 7.0, -INF], len(ids)))})
    return rep, freq, pres, hists, bias


def open_rows(eng, rep, freq, pres, hists, bias, last_n=-1, penalty_from=0, **kw):
    p = fb.make_params(len(rep), repeat_last_n=last_n, penalty_from=penalty_from, seed=1, **kw)
    p["repetition_penalty"] = rep
    p["seed"] = 11 + np.arange(len(rep))
    sids = eng.open_streams(p)
    for r, sid in enumerate(sids):
        eng.history_set(int(sid), hists[r])
        eng.set_penalties(int(sid), freq[r], pres[r])
        eng.set_bias(int(sid), bias[r])
    return sids


def engine_for(rows, V, ids=1 << 20):
    e = fb.Engine(device=0, max_rows=rows, max_vocab=V, max_hist_ids=ids)
    e.set_cuda_stream(torch.cuda.current_stream().cuda_stream)
    return e


@pytest.mark.parametrize("rows,V,pad,out_pad,shift,in_t,out_t,cap,hist,n_bias", [
    (1, 1, 0, 0, 0, "f32", "f32", 0.0, 3, 1),
    (1, 31, 0, 0, 0, "bf16", "f32", 0.0, 40, 5),
    (3, 33, 1, 2, 1, "f16", "f16", 30.0, 40, 5),
    (5, 4095, 1, 0, 0, "f32", "f32", 0.0, 300, 20),
    (2, 4096, 0, 0, 0, "bf16", "bf16", 0.0, 300, 0),
    (4, 4097, 7, 7, 0, "f16", "f32", 0.0, 0, 20),
    (17, 8200, 0, 0, 0, "f32", "f32", 30.0, 1000, 300),
    (9, 20000, 8, 4, 0, "bf16", "f32", 5.0, 6000, 40),
    (97, 5003, 5, 9, 1, "bf16", "f32", 0.0, 100, 10),
    (513, 1000, 0, 0, 0, "f32", "f32", 0.0, 60, 4),
    (2, 262144, 0, 0, 0, "f32", "f32", 30.0, 30000, 300),
])
def test_against_64_bits(rows, V, pad, out_pad, shift, in_t, out_t, cap, hist, n_bias):
    rng = np.random.default_rng(V + rows)
    buf = torch.zeros(rows * (V + pad) + shift + 64, dtype=T[in_t], device="cuda")
    logits = buf[shift:shift + rows * (V + pad)].view(rows, V + pad)
    logits.copy_(torch.from_numpy(rng.standard_normal((rows, V + pad)).astype(np.float32) * 6))
    rep, freq, pres, hists, bias = settings(rng, rows, V, hist, n_bias)
    allowed = [None if r % 4 == 3 else rng.random(V) < [0.5, 0.002, 0.98][r % 4] for r in range(rows)]
    if rows > 2:
        allowed[2] = np.zeros(V, dtype=bool)                   # nothing is left
    which = np.full(rows, -1, dtype=np.int32)
    order = [r for r in rng.permutation(rows) if allowed[r] is not None]
    which[order] = np.arange(len(order))
    words = (V + 31) // 32
    masks = pack([allowed[r] for r in order], words) if order else None
    for r in range(rows):                                      # what lies where a mask forbids does not matter
        if allowed[r] is not None:
            logits[r, :V][torch.from_numpy(~allowed[r]).cuda()] = [float("nan"), INF, -INF, torch.finfo(T[in_t]).min][r % 4]
    eng = engine_for(rows, V)
    eng.set_softcap(cap)
    sids = open_rows(eng, rep, freq, pres, hists, bias)
    want, mag = plain(logits, V, hists, rep, freq, pres, bias, allowed, cap)
    # the result stands in the middle of a larger buffer, which stays as it was
    frame = torch.full((rows + 2, V + out_pad + 3), 7.0, dtype=T[out_t], device="cuda")
    out = frame[1:rows + 1, 1 if out_pad else 0:][:, :V + (out_pad if out_pad else 0)]
    before = frame.clone()
    r = eng.adjust_logits(sids, logits, out, masks=masks, mask_rows=which, n_vocab=V)
    torch.cuda.synchronize()
    assert r is out
    check(out[:, :V], want, mag, cap, out_t)
    out[:, :V] = 7.0
    assert torch.equal(frame, before)
    # in place
    if in_t == out_t:
        tail = logits[:, V:].clone()
        eng.adjust_logits(sids, logits, logits, masks=masks, mask_rows=which, n_vocab=V)
        check(logits[:, :V], want, mag, cap, out_t)
        assert torch.equal(logits[:, V:], tail) or V + pad == V
    eng.close()


@pytest.mark.parametrize("last_n,penalty_from", [(-1, 0), (0, 0), (5, 0), (1, 0), (1000, 0), (-1, 7), (6, 18), (-1, 20), (-1, 500)])
def test_the_window_is_the_repetition_penaltys(last_n, penalty_from):
    rng = np.random.default_rng(3)
    V, hist = 300, rng.integers(0, 30, 20).astype(np.int32)
    logits = torch.from_numpy(rng.standard_normal((1, V)).astype(np.float32) * 3).cuda()
    b = 0 if last_n < 0 or last_n >= 20 else 20 - last_n
    window = hist[max(b, penalty_from):] if last_n != 0 else hist[:0]
    for rep in (1.0, 1.3):    # frequency and presence have their window without a repetition penalty, too
        eng = engine_for(1, V)
        sids = open_rows(eng, [rep], [0.5], [0.25], [hist], [{}], last_n=last_n, penalty_from=penalty_from)
        out = eng.adjust_logits(sids, logits, torch.empty_like(logits))
        want, mag = plain(logits, V, [window], [rep], [0.5], [0.25], [{}], [None], 0.0)
        check(out, want, mag, 0.0, "f32")
        eng.close()


@pytest.mark.parametrize("in_t", ["f32", "bf16", "f16"])
def test_special_values(in_t):
    """Infinities, NaN, zeros and the ends of the type, allowed and penalised."""
    f = torch.finfo(T[in_t])
    vals = [INF, -INF, float("nan"), 0.0, -0.0, f.max, f.min, f.tiny, -f.tiny, f.smallest_normal, 1.0, -1.0]
    V = 2 * len(vals)
    logits = torch.tensor([vals + vals], device="cuda").to(T[in_t])
    hist = np.arange(len(vals), dtype=np.int32)
    eng = engine_for(1, V)
    sids = open_rows(eng, [1.5], [0.5], [0.25], [hist], [{}])
    out = eng.adjust_logits(sids, logits, torch.empty(1, V, device="cuda"))
    x = logits.float().cpu().numpy()[0]
    with np.errstate(over="ignore", invalid="ignore"):
        y = x.copy()
        n = len(vals)
        y[:n] = np.where(x[:n] > 0, x[:n] / np.float32(1.5), x[:n] * np.float32(1.5)) - np.float32(0.75)
    assert np.array_equal(out.cpu().numpy()[0], y, equal_nan=True)
    # an infinite bias is a ban, whatever it is added to
    eng.set_bias(int(sids[0]), {0: -INF, 1: -INF, 2: -INF, 10: 2.0})
    out = eng.adjust_logits(sids, logits, out)
    y[:3] = -INF
    y[10] += np.float32(2.0)
    assert np.array_equal(out.cpu().numpy()[0], y, equal_nan=True)
    eng.close()


@pytest.mark.parametrize("cap", [1e-12, 0.5, 30.0, 1e12])
def test_softcap_over_its_range(cap):
    """Relative error: with a = 2 x / cap, e^a is within 2^-22 and its argument's rounding, the reciprocal within 2^-23; 2 / (e^a + 1) is 0.66 where the
    result is smallest, 0.34: below 1.7 * 2^-21 with the sums' roundings, 2^-23 for the division and the product by cap: 2^-20 in all.  Quotients
    below the smallest normal number are off by 2^-149."""
    cap = float(np.float32(cap))
    f = torch.finfo(torch.float32)
    u = np.concatenate([np.linspace(-12, 12, 20001), np.linspace(-0.4, 0.4, 4001), 10.0 ** np.linspace(-30, 0, 61)]) * cap
    vals = np.concatenate([u, [INF, -INF, float("nan"), 0.0, -0.0, f.max, f.min, f.tiny, -f.tiny, 1.0, -1.0]]).astype(np.float32)
    logits = torch.from_numpy(vals[None]).cuda()
    eng = engine_for(1, len(vals))
    eng.set_softcap(cap)
    sid = eng.open_stream(fb.make_params(1, repetition_penalty=1.0, seed=1))
    got = eng.adjust_logits([sid], logits, torch.empty_like(logits)).cpu().numpy()[0].astype(np.float64)
    want = cap * np.tanh(vals.astype(np.float64) / cap)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    worst = np.abs(got[ok] - want[ok]) - (2.0 ** -20 * np.abs(want[ok]) + 2.0 ** -149 * max(cap, 1.0))
    assert worst.max() <= 0, vals[ok][np.argmax(worst)]
    eng.close()


@pytest.mark.parametrize("rows,in_t", [(1, "f32"), (3, "bf16")])
def test_windows_of_more_than_65535_ids(rows, in_t):
    """Counts that 16 bits do not hold, and windows whose ids fall into all tiles."""
    rng = np.random.default_rng(12)
    V, n = 20003, 70001
    hists = [np.full(n, 7, dtype=np.int32), rng.integers(0, V, 65536).astype(np.int32), rng.integers(0, V, 65535).astype(np.int32)][:rows]
    hists[0][-5:] = [7, V - 1, 7, 4096, 0]
    logits = torch.from_numpy(rng.standard_normal((rows, V)).astype(np.float32) * 4).cuda().to(T[in_t])
    rep, freq, pres, bias = [1.3] * rows, [0.001, 0.25, -0.5][:rows], [0.5] * rows, [{7: 2.0, V - 1: -1.0}] * rows
    eng = engine_for(rows, V)
    sids = open_rows(eng, rep, freq, pres, hists, bias)
    want, mag = plain(logits, V, hists, rep, freq, pres, bias, [None] * rows, 0.0)
    out = eng.adjust_logits(sids, logits, torch.empty(rows, V, device="cuda"))
    check(out, want, mag, 0.0, "f32")
    eng.close()


@pytest.mark.parametrize("in_t,out_t", [("bf16", "f32"), ("f16", "f16")])
def test_rows_that_are_gigabytes_apart(in_t, out_t):
    """Row offsets beyond 2^31 elements, and masks beyond 2^31 words' bytes."""
    rng = np.random.default_rng(15)
    V, ld, rows = 5000, 1 << 30, 3
    logits = torch.empty(2 * ld + V, dtype=T[in_t], device="cuda").as_strided((rows, V), (ld, 1))
    logits.copy_(torch.from_numpy(rng.standard_normal((rows, V)).astype(np.float32) * 4))
    out = torch.empty(2 * ld + V, dtype=T[out_t], device="cuda").as_strided((rows, V), (ld, 1))
    allowed = [rng.random(V) < 0.5 for _ in range(rows)]
    words = (V + 31) // 32
    masks = torch.empty(ld + words, dtype=torch.int32, device="cuda").as_strided((rows, words), (ld // 2, 1))
    masks.copy_(pack(allowed, words))
    eng = engine_for(rows, V)
    rep, freq, pres, hists, bias = settings(rng, rows, V, 400, 30)
    sids = open_rows(eng, rep, freq, pres, hists, bias)
    want, mag = plain(logits, V, hists, rep, freq, pres, bias, allowed, 0.0)
    eng.adjust_logits(sids, logits, out, masks=masks)
    check(out, want, mag, 0.0, out_t)
    eng.close()


@pytest.mark.parametrize("offset", [0, 1, 31, 32, 5000])
def test_vocabulary_shards(offset):
    rng = np.random.default_rng(offset)
    rows, V = 4, 3001
    logits = torch.from_numpy(rng.standard_normal((rows, V)).astype(np.float32) * 3).cuda()
    rep, freq, pres, hists, bias = settings(rng, rows, V, 200, 50, offset)
    allowed = [rng.random(V) < 0.5 for _ in range(rows)]
    words = (offset + V + 31) // 32
    eng = engine_for(rows, V)
    eng.set_vocab_offset(offset)
    sids = open_rows(eng, rep, freq, pres, hists, bias)
    out = eng.adjust_logits(sids, logits, torch.empty_like(logits), masks=pack(allowed, words, offset))
    want, mag = plain(logits, V, hists, rep, freq, pres, bias, allowed, 0.0, offset)
    check(out, want, mag, 0.0, "f32")
    eng.close()


def test_settings_come_and_go_with_their_stream():
    V = 512
    rng = np.random.default_rng(1)
    logits = torch.from_numpy(rng.standard_normal((1, V)).astype(np.float32)).cuda()
    out = torch.empty_like(logits)
    eng = engine_for(1, V, ids=1024)   # four regions of the smallest size
    for _ in range(40):                # regions are given back
        sids = open_rows(eng, [1.2], [0.5], [0.0], [[1, 2, 2]], [{5: 3.0, 9: -2.0}])
        eng.adjust_logits(sids, logits, out)
        want, mag = plain(logits, V, [[1, 2, 2]], [1.2], [0.5], [0.0], [{5: 3.0, 9: -2.0}], [None], 0.0)
        check(out, want, mag, 0.0, "f32")
        for n in (1, 100, 200, 3):     # lists that grow out of their region and shrink
            b = {i: float(i % 7) - 3.0 for i in range(n)}
            eng.set_bias(int(sids[0]), b)
            eng.adjust_logits(sids, logits, out)
            want, mag = plain(logits, V, [[1, 2, 2]], [1.2], [0.5], [0.0], [b], [None], 0.0)
            check(out, want, mag, 0.0, "f32")
        eng.close_stream(int(sids[0]))
        again = eng.open_stream(fb.make_params(1, repetition_penalty=1.0, seed=1))   # the id is used again, its settings are not
        assert again == sids[0]
        assert torch.equal(eng.adjust_logits([again], logits, out), logits)
        eng.close_stream(again)
    # a list that the pool cannot hold leaves the old one in force
    sid = eng.open_stream(fb.make_params(1, repetition_penalty=1.0, seed=1))
    eng.set_bias(sid, {7: 1.0})
    with pytest.raises(fb.SamplerError) as e:
        eng.set_bias(sid, {i: 1.0 for i in range(600)})
    assert e.value.code == -3
    eng.adjust_logits([sid], logits, out)
    assert float(out[0, 7]) == float(logits[0, 7] + 1.0)
    eng.set_bias(sid, {})
    assert torch.equal(eng.adjust_logits([sid], logits, out), logits)
    eng.close()


def test_settings_that_change_while_calls_are_queued():
    """A call sees the settings of its moment, however late it runs: histories, biases and regions that change hands behind it."""
    rng = np.random.default_rng(9)
    V = 3000
    logits = torch.from_numpy(rng.standard_normal((1, V)).astype(np.float32) * 3).cuda()
    eng = engine_for(1, V, ids=2048)
    big = torch.zeros(1 << 27, device="cuda")
    outs, wants = [], []
    torch.cuda.synchronize()
    for _ in range(12):
        big.add_(1.0)                                    # everything below is queued behind this
        hist = rng.integers(0, 40, int(rng.integers(1, 500))).astype(np.int32)
        bias = {int(i): 1.5 for i in rng.permutation(V)[: int(rng.integers(1, 200))]}
        sid = int(open_rows(eng, [1.3], [0.25], [0.5], [hist], [bias])[0])
        for step in range(3):
            out = torch.empty_like(logits)
            eng.adjust_logits([sid], logits, out)
            outs.append(out)
            wants.append(plain(logits, V, [hist], [1.3], [0.25], [0.5], [bias], [None], 0.0))
            if step == 0:
                bias = {int(i): -2.0 for i in rng.permutation(V)[:150]}
                eng.set_bias(sid, bias)
            else:
                hist = rng.integers(0, 40, 300).astype(np.int32)
                eng.history_set(sid, hist)
        eng.close_stream(sid)                            # its regions are the next one's
    torch.cuda.synchronize()
    for out, (want, mag) in zip(outs, wants):
        check(out, want, mag, 0.0, "f32")
    eng.close()


def test_one_stream_for_several_rows_and_another_cuda_stream():
    rng = np.random.default_rng(8)
    V, rows = 9000, 6
    logits = torch.from_numpy(rng.standard_normal((rows, V)).astype(np.float32) * 3).cuda()
    eng = fb.Engine(device=0, max_rows=rows, max_vocab=V, max_hist_ids=1 << 16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    eng.set_cuda_stream(side.cuda_stream)
    hist = rng.integers(0, V, 700).astype(np.int32)
    sid = int(open_rows(eng, [1.4], [0.2], [0.1], [hist], [{3: 4.0}])[0])
    out = torch.empty_like(logits)
    torch.cuda.current_stream().synchronize()
    for _ in range(5):
        eng.adjust_logits([sid] * rows, logits, out)
    side.synchronize()
    want, mag = plain(logits, V, [hist] * rows, [1.4] * rows, [0.2] * rows, [0.1] * rows, [{3: 4.0}] * rows, [None] * rows, 0.0)
    check(out, want, mag, 0.0, "f32")
    eng.close()


def test_refusals():
    V, rows = 1000, 2
    eng = engine_for(rows, V, ids=4096)
    sids = eng.open_streams(fb.make_params(rows, seed=1))
    lg = torch.zeros(rows, V, device="cuda")
    out = torch.empty_like(lg)
    masks = torch.zeros(rows, 32, dtype=torch.int32, device="cuda")

    def code(**kw):
        a = dict(sids=sids, logits=lg, out=out, masks=masks, mask_rows=None)
        a.update(kw)
        with pytest.raises(fb.SamplerError) as e:
            eng.adjust_logits(a["sids"], a["logits"], a["out"], masks=a["masks"], mask_rows=a["mask_rows"])
        return e.value.code

    assert code(sids=[0, 77]) == -5
    assert code(masks=masks[:, :31].contiguous()) == -1
    assert code(masks=masks[:1]) == -1
    assert code(mask_rows=[0, 2]) == -1 and code(mask_rows=[-2, 0]) == -1
    assert code(masks=None, mask_rows=[0, -1]) == -1
    assert code(out=out.to(torch.bfloat16)) == -1
    assert code(logits=lg.to(torch.bfloat16), out=out.to(torch.float16)) == -1
    both = torch.zeros(rows * V + 8, device="cuda")
    assert code(logits=both[:rows * V].view(rows, V), out=both[4:4 + rows * V].view(rows, V)) == -1
    big = torch.zeros(3, V, device="cuda")
    assert code(sids=[0, 0, 0], logits=big, out=torch.empty_like(big), masks=None) == -3
    wide = torch.zeros(rows, V + 1, device="cuda")
    assert code(logits=wide, out=torch.empty_like(wide), masks=None) == -3
    for bad in (dict(logits=lg.double()), dict(masks=masks.long())):
        with pytest.raises(TypeError):
            eng.adjust_logits(sids, bad.get("logits", lg), out, masks=bad.get("masks", masks))
    for bad in (dict(logits=lg.cpu()), dict(masks=masks.cpu()), dict(logits=torch.zeros(V, rows, device="cuda").T), dict(sids=[0]), dict(out=out[:, :5])):
        with pytest.raises(ValueError):
            eng.adjust_logits(bad.get("sids", sids), bad.get("logits", lg), bad.get("out", out), masks=bad.get("masks", masks))
    with pytest.raises(ValueError):
        eng.adjust_logits(sids, lg, out, masks=masks, mask_rows=[0])
    for f, p in ((float("nan"), 0.0), (0.0, INF)):
        with pytest.raises(fb.SamplerError) as e:
            eng.set_penalties(0, f, p)
        assert e.value.code == -2
    for ids, v, want in (([1, 2, 1], [0.0, 0.0, 1.0], -1), ([1], [INF], -2), ([1], [float("nan")], -2)):
        with pytest.raises(fb.SamplerError) as e:
            eng.set_bias(0, ids, v)
        assert e.value.code == want
    # not inside a capture
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    eng.set_cuda_stream(s.cuda_stream)
    with torch.cuda.graph(g, stream=s):
        lg.add_(0.0)
        with pytest.raises(fb.SamplerError) as e:
            eng.adjust_logits(sids, lg, out)
        assert e.value.code == -1
    # and the engine goes on as before
    eng.adjust_logits(sids, lg, out, masks=masks)
    s.synchronize()
    assert bool(torch.isneginf(out).all())
    eng.close()
