"""From hidden states to tokens: the LM head, the adjustment and the sampler together, as a decode loop uses them."""
import numpy as np
import pytest

import ferro_b200 as fb

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_adjust_gpu import open_rows, pack, plain as plain_adjust, settings  # noqa: E402
from test_head_gpu import integers, plain as plain_head  # noqa: E402

INF = float("inf")


def engine_for(rows, V, ids=1 << 18):
    e = fb.Engine(device=0, max_rows=rows, max_vocab=V, max_hist_ids=ids)
    e.set_cuda_stream(torch.cuda.current_stream().cuda_stream)
    return e


def test_a_decode_loop_from_hidden_states(oracle):
    """Eight streams of different requests, twelve steps.  Logits are exact (integers), so that the oracle, which draws from the
    float32 rows that the adjustment leaves, must give the same tokens."""
    rng = np.random.default_rng(12)
    rows, V, K = 8, 3000, 256
    w, s, _ = integers(rng, rows, V, K, 64, "f16", "bf16")
    s = torch.full_like(s, 0.03125)
    eng, twin = engine_for(rows, V), engine_for(rows, V)
    heads = [e.load_head(w, s) for e in (eng, twin)]
    rep, freq, pres, hists, bias = settings(rng, rows, V, 60, 20)
    hists = [np.clip(h, 0, V - 1) for h in hists]
    kw = dict(temperature=0.8, top_k=40, top_p=0.95)
    ids = [open_rows(e, rep, freq, pres, hists, bias, **kw) for e in (eng, twin)]
    p = fb.make_params(rows, repetition_penalty=1.0, **kw)
    p["seed"] = 11 + np.arange(rows)
    rngs = oracle.new_rngs(p["seed"])
    grown = [list(h) for h in hists]
    for step in range(12):
        x = torch.from_numpy(rng.integers(-7, 8, (rows, K)).astype(np.float32)).to(torch.bfloat16).cuda()
        allowed = [rng.random(V) < 0.3 for _ in range(rows)]
        which = np.arange(rows, dtype=np.int32)
        which[step % rows] = -1
        masks = pack(allowed, (V + 31) // 32)
        # in one call
        tok = eng.sample_hidden(heads[0], ids[0], x, masks=masks, mask_rows=which, flags=fb.APPEND_SAMPLED)
        # in three
        lg = heads[1].logits(x, torch.empty(rows, V, device="cuda"))
        assert torch.equal(lg.double(), plain_head(w, s, x))
        adj = twin.adjust_logits(ids[1], lg, torch.empty_like(lg), masks=masks, mask_rows=which)
        torch.cuda.synchronize()
        tok2 = twin.sample_batch_adjusted(ids[1], lg, masks=masks, mask_rows=which, flags=fb.APPEND_SAMPLED)
        ref = oracle.sample_rows(p, rngs, adj.cpu().numpy().copy(), [[]] * rows)
        assert np.array_equal(tok, tok2) and np.array_equal(tok, ref["tokens"]), step
        want, _ = plain_adjust(lg, V, grown, rep, freq, pres, bias, [None if which[r] < 0 else allowed[r] for r in range(rows)], 0.0)
        assert np.allclose(adj.cpu().numpy(), want, rtol=0, atol=2.0 ** -24 * 6 * 200)   # (magnitudes below 200)
        for r in range(rows):
            assert which[r] < 0 or allowed[r][tok[r]]
            assert bias[r].get(int(tok[r]), 0.0) != -INF
            grown[r].append(int(tok[r]))
            assert eng.history_len(int(ids[0][r])) == len(grown[r])
    assert [eng.stream_state(int(i)) for i in ids[0]] == [twin.stream_state(int(i)) for i in ids[1]]
    eng.close()
    twin.close()


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("in_t", [torch.float32, torch.bfloat16])
def test_without_extras_the_adjusted_call_is_the_resident_call(cap, in_t):
    rng = np.random.default_rng(21)
    rows, V = 6, 5001
    lg = torch.from_numpy(rng.standard_normal((rows, V)).astype(np.float32) * 4).cuda().to(in_t)
    hists = [rng.integers(0, V, 200).astype(np.int32) for _ in range(rows)]
    got = []
    for k in range(2):
        e = engine_for(rows, V)
        e.set_softcap(cap)
        sids = open_rows(e, np.full(rows, 1.3, np.float32), [0.0] * rows, [0.0] * rows, hists, [{}] * rows, temperature=0.7, top_k=30)
        toks = []
        for _ in range(6):
            if k == 0:
                toks.append(e.sample_batch_adjusted(sids, lg, flags=fb.APPEND_SAMPLED))
            else:
                full = lg.float()
                toks.append(e.sample_batch_resident(sids, full.data_ptr(), n_vocab=V, flags=fb.APPEND_SAMPLED))
        got.append(np.array(toks))
        e.close()
    assert np.array_equal(got[0], got[1])


@pytest.mark.parametrize("mode", [0, 1, 2])
def test_overlapping_launches_read_fresh_rows(mode):
    """Whatever the launch mode, sampling waits for the head and the adjustment."""
    rng = np.random.default_rng(33)
    rows, V, K = 64, 20000, 64
    w, s, x = integers(rng, rows, V, K, 32, "f16", "bf16")
    e = engine_for(rows, V)
    e.set_launch_overlap(mode)
    head = e.load_head(w, s)
    p = fb.make_params(rows, temperature=0.0, repetition_penalty=1.0)
    p["seed"] = 1
    sids = e.open_streams(p)
    for _ in range(20):
        x = torch.from_numpy(rng.integers(-7, 8, (rows, K)).astype(np.float32)).to(torch.bfloat16).cuda()
        lg = plain_head(w, s, x)
        best = (lg == lg.max(dim=1, keepdim=True).values).float().argmax(dim=1).cpu().numpy()   # the lowest of equals
        assert np.array_equal(e.sample_hidden(head, sids, x), best)
        allowed = rng.random((rows, V)) < 0.01
        allowed[:, 5] = True
        lg = torch.where(torch.from_numpy(allowed).cuda(), lg, -INF)
        best = (lg == lg.max(dim=1, keepdim=True).values).float().argmax(dim=1).cpu().numpy()
        assert np.array_equal(e.sample_hidden(head, sids, x, masks=pack(allowed, (V + 31) // 32)), best)
    e.close()


@pytest.mark.parametrize("rows,V,top_k,temperature", [(3, 100, 0, 1.0), (5, 9000, 40, 0.8), (70, 4097, 50, 0.0), (4, 70000, 300, 0.9)])
def test_a_row_that_nothing_is_left_of_ends_the_call(rows, V, top_k, temperature):
    rng = np.random.default_rng(V)
    lg = torch.from_numpy(rng.standard_normal((rows, V)).astype(np.float32)).cuda()
    e = engine_for(rows, V)
    sids = open_rows(e, np.full(rows, 1.1, np.float32), [0.1] * rows, [0.0] * rows, [[1, 2, 3]] * rows, [{}] * rows, temperature=temperature, top_k=top_k)
    allowed = np.zeros((rows, V), dtype=bool)
    allowed[:, [1, V // 2, V - 1]] = True
    full = pack(allowed, (V + 31) // 32)
    allowed[rows - 1] = False
    empty = pack(allowed, (V + 31) // 32)
    state = [e.stream_state(int(i)) for i in sids]
    for _ in range(3):
        with pytest.raises(fb.SamplerError) as err:
            e.sample_batch_adjusted(sids, lg, masks=empty, flags=fb.APPEND_SAMPLED)
        assert err.value.code == -8 and f"row {rows - 1} " in str(err.value)
        assert [e.stream_state(int(i)) for i in sids] == state and all(e.history_len(int(i)) == 3 for i in sids)
    # a row whose only tokens are banned by their biases is as empty
    e.set_bias(int(sids[0]), {1: -INF, V // 2: -INF, V - 1: -INF})
    with pytest.raises(fb.SamplerError) as err:
        e.sample_batch_adjusted(sids, lg, masks=full)
    assert err.value.code == -8 and "row 0 " in str(err.value)
    e.set_bias(int(sids[0]), {})
    tok = e.sample_batch_adjusted(sids, lg, masks=full, flags=fb.APPEND_SAMPLED)
    assert all(t in (1, V // 2, V - 1) for t in tok) and all(e.history_len(int(i)) == 4 for i in sids)
    e.close()


def test_refusals():
    rows, V, K = 2, 500, 64
    rng = np.random.default_rng(1)
    w, s, x = integers(rng, rows, V, K, 32, "f16", "bf16")
    e = engine_for(rows, V)
    head = e.load_head(w, s)
    sids = e.open_streams(fb.make_params(rows, seed=3))
    lg = torch.zeros(rows, V, device="cuda")

    def code(f):
        with pytest.raises(fb.SamplerError) as err:
            f()
        return err.value.code

    for call in (lambda ids, **kw: e.sample_batch_adjusted(ids, lg, **kw), lambda ids, **kw: e.sample_hidden(head, ids, x, **kw)):
        assert code(lambda: call([0, 0])) == -1
        assert code(lambda: call([0, 9])) == -5
        for flags in (fb.WRITE_BACK, fb.LOGITS_ON_HOST, 64):
            assert code(lambda: call(sids, flags=flags)) == -1
        with pytest.raises(ValueError):
            call([0])
        e.set_vocab_shard(0, 2 * V)
        assert code(lambda: call(sids)) == -1
        e.set_vocab_shard(0, 0)
    small = engine_for(rows, V - 1)
    big = small.load_head(w, s)
    small.open_streams(fb.make_params(rows, seed=3))
    assert code(lambda: small.sample_hidden(big, [0, 1], x)) == -3
    assert e.stream_state(int(sids[0]))[1] == 0
    small.close()
    e.close()
