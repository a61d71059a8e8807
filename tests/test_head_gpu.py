"""The LM head with 4-bit weights (fsb_head_*) against a plain implementation in 64 bits.

Where hidden states are small integers and scales powers of two, every sum is an integer multiple of a power of two below 2^24
of it, so that fp32 holds it exactly in any order: the logits must then be equal, bit for bit.  Else: products are exact; per
group of n weights the kernel adds up n products of at most 31 |x| on top of 24 times the group's sum of x, each of these n + 1 additions
off by at most 2^-23 (tensor cores may cut off) of what has been added up, at most 55 S with S the sum of |x| over the group, and the sum
of x itself by n 2^-24 S, times 24; scales and the sum over groups add 2^-24 (groups + 20) of the sum of |scale| times at most 55 S."""
import numpy as np
import pytest

import ferro_b200 as fb

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def unpack(w):
    return torch.stack([w & 15, w >> 4], dim=2).view(w.shape[0], -1).double() - 8.0


def plain(w, s, x):
    W = unpack(w) * s.double().repeat_interleave(2 * w.shape[1] // s.shape[1], dim=1)
    return x.double() @ W.T


def engine():
    e = fb.Engine(device=0, max_rows=64, max_vocab=1 << 16, max_hist_ids=1 << 16)
    e.set_cuda_stream(torch.cuda.current_stream().cuda_stream)
    return e


def integers(rng, rows, V, K, group, scale_t, hidden_t):
    w = torch.from_numpy(rng.integers(0, 256, (V, K // 2), dtype=np.uint8)).cuda()
    s = torch.from_numpy(2.0 ** rng.integers(-2, 2, (V, K // group))).float().to(T[scale_t]).cuda()
    x = torch.from_numpy(rng.integers(-7, 8, (rows, K)).astype(np.float32)).to(T[hidden_t]).cuda()
    return w, s, x


@pytest.mark.parametrize("rows,V,K,group,scale_t,hidden_t,pad,out_pad", [
    (1, 1, 32, 32, "f16", "bf16", 0, 0),
    (1, 33, 64, 32, "bf16", "f16", 0, 3),
    (2, 31, 96, 32, "f16", "bf16", 1, 0),
    (3, 500, 128, 64, "f16", "f16", 0, 1),
    (7, 1000, 256, 128, "bf16", "bf16", 8, 0),
    (8, 129, 384, 128, "f16", "f16", 3, 0),
    (8, 2049, 2016, 32, "f16", "bf16", 0, 0),
    (9, 513, 1024, 32, "bf16", "f16", 0, 4),
    (15, 777, 192, 64, "bf16", "bf16", 0, 0),
    (16, 5000, 2560, 64, "f16", "bf16", 0, 0),
    (17, 300, 2048, 128, "f16", "f16", 8, 0),
    (24, 1500, 608, 32, "bf16", "bf16", 0, 0),
    (31, 4097, 1120, 32, "f16", "f16", 0, 1),
    (32, 640, 2560, 128, "bf16", "bf16", 0, 0),
    (33, 1000, 512, 32, "f16", "bf16", 0, 0),
    (64, 3000, 2560, 32, "f16", "bf16", 0, 0),
    (65, 260, 320, 64, "bf16", "f16", 2, 0),
    (129, 1111, 1024, 64, "f16", "f16", 0, 0),
    (136, 700, 2048, 32, "f16", "bf16", 0, 0),
    (300, 450, 640, 128, "bf16", "bf16", 0, 5),
    (4, 20000, 96, 32, "f16", "bf16", 0, 0),
    (40, 20000, 64, 64, "f16", "bf16", 0, 0),
    (10, 700, 1280, 128, "bf16", "f16", 0, 0),
    (12, 2050, 448, 64, "f16", "bf16", 1, 0),
    (33, 777, 1056, 32, "bf16", "bf16", 1, 0),
    (64, 1025, 2048, 64, "f16", "f16", 3, 2),
    (97, 300, 896, 128, "f16", "bf16", 8, 0),
    (144, 513, 1024, 32, "f16", "bf16", 0, 0),
    (145, 600, 576, 64, "bf16", "f16", 0, 0),
    (64, 40000, 96, 32, "f16", "bf16", 0, 0),
    (65, 77777, 32, 32, "f16", "bf16", 0, 0),
])
def test_exact_sums_are_exact(rows, V, K, group, scale_t, hidden_t, pad, out_pad):
    rng = np.random.default_rng(rows * 1000 + K)
    w, s, x = integers(rng, rows, V, K, group, scale_t, hidden_t)
    xp = torch.full((rows, K + pad), float("nan"), dtype=T[hidden_t], device="cuda")
    xp[:, :K] = x
    e = engine()
    head = e.load_head(w, s)
    frame = torch.full((rows + 2, V + out_pad), 7.0, device="cuda")
    out = frame[1:rows + 1, :V]
    assert head.logits(xp[:, :K], out) is out
    assert torch.equal(out.double(), plain(w, s, x))
    assert bool((frame[0] == 7).all()) and bool((frame[-1] == 7).all()) and bool((frame[:, V:] == 7).all())
    e.close()


@pytest.mark.parametrize("rows,V,K,group", [(1, 300, 16384, 32), (6, 200, 16384, 128), (13, 300, 8192, 64), (50, 150, 16384, 32), (200, 260, 8192, 32)])
def test_long_rows(rows, V, K, group):
    """Hidden states that do not all fit shared memory at once; values whose sums stay below 2^24."""
    rng = np.random.default_rng(K + rows)
    w, s, x = integers(rng, rows, V, K, group, "f16", "bf16")
    e = engine()
    out = e.load_head(w, s).logits(x, torch.empty(rows, V, device="cuda"))
    assert torch.equal(out.double(), plain(w, s, x))
    e.close()


@pytest.mark.parametrize("rows", [1, 8, 16, 40, 130])
@pytest.mark.parametrize("group,scale_t,hidden_t", [(32, "f16", "bf16"), (64, "bf16", "f16"), (128, "f16", "f16")])
def test_against_64_bits(rows, group, scale_t, hidden_t):
    rng = np.random.default_rng(rows + group)
    V, K = 1000, 1280
    w = torch.from_numpy(rng.integers(0, 256, (V, K // 2), dtype=np.uint8)).cuda()
    s = torch.from_numpy((0.5 + rng.random((V, K // group))) * 0.02).to(T[scale_t]).cuda()
    s[::7] *= -1.0
    x = torch.from_numpy(rng.standard_normal((rows, K)) * np.exp(2 * rng.standard_normal((1, K)))).to(T[hidden_t]).cuda()
    e = engine()
    out = e.load_head(w, s).logits(x, torch.empty(rows, V, device="cuda"))
    want = plain(w, s, x)
    S = x.double().abs().view(rows, -1, group).sum(2)                # [rows][groups]
    scaled = (S @ s.double().abs().T) * 55
    tol = scaled * ((group + 1) * 2.0 ** -23 + 24 / 55 * group * 2.0 ** -24 + (K // group + 20) * 2.0 ** -24)
    assert bool(((out.double() - want).abs() <= tol).all())
    # and as a whole about as exact as fp32 sums are: each of the errors above is one of many of either sign
    rel = float((out.double() - want).norm() / want.norm())
    assert rel <= 55 / 4.6 * 2.0 ** -23, rel     # 4.6: the root mean square of q - 8
    e.close()


def test_infinite_and_nan_hidden_states_stay_in_their_rows():
    rng = np.random.default_rng(2)
    for rows in (3, 40):
        w, s, x = integers(rng, rows, 300, 256, 32, "f16", "bf16")
        x[1, 5] = float("nan")
        x[2, 7] = float("inf")
        e = engine()
        out = e.load_head(w, s).logits(x, torch.empty(rows, 300, device="cuda"))
        clean = [r for r in range(rows) if r not in (1, 2)]
        assert torch.equal(out[clean].double(), plain(w, s, x[clean])) and not bool(torch.isfinite(out[1:3]).any())
        e.close()


@pytest.mark.parametrize("rows", [2, 20])
def test_weights_and_rows_beyond_four_gigabytes(rows):
    """4.7 GB of weights, laid out and multiplied; hidden states and logits whose rows are gigabytes apart."""
    V, K, group, ld = 575000, 16384, 128, (1 << 30) // 8
    torch.manual_seed(rows)
    w = torch.randint(0, 256, (V, K // 2), dtype=torch.uint8, device="cuda")
    s = (2.0 ** torch.randint(-2, 2, (V, K // group), device="cuda")).to(torch.bfloat16)
    x = torch.empty((rows - 1) * ld + K, dtype=torch.bfloat16, device="cuda").as_strided((rows, K), (ld, 1))
    x.copy_(torch.randint(-7, 8, (rows, K), device="cuda"))
    out = torch.empty((rows - 1) * ld + V, dtype=torch.float32, device="cuda").as_strided((rows, V), (ld, 1))
    e = fb.Engine(device=0, max_rows=32, max_vocab=1 << 20, max_hist_ids=1 << 16)
    e.set_cuda_stream(torch.cuda.current_stream().cuda_stream)
    head = e.load_head(w, s)
    head.logits(x, out)
    for at in (0, 262100, 524200, V - 300):      # (2^32 bytes of weights end at row 524288)
        assert torch.equal(out[:, at:at + 300].double(), plain(w[at:at + 300], s[at:at + 300], x)), at
    e.close()


def test_weights_may_come_from_the_host_and_go_away():
    rng = np.random.default_rng(4)
    w, s, x = integers(rng, 5, 777, 160, 32, "bf16", "f16")
    e = engine()
    wh, sh = w.cpu(), s.cpu()
    head = e.load_head(wh, sh)
    wh.zero_(), sh.zero_()
    other = e.load_head(w, s)
    w2, s2 = w.clone(), s.clone()
    w.zero_(), s.zero_()
    a, b = torch.empty(5, 777, device="cuda"), torch.empty(5, 777, device="cuda")
    head.logits(x, a), other.logits(x, b)
    assert torch.equal(a.double(), plain(w2, s2, x)) and torch.equal(a, b)
    head.free()
    with pytest.raises(fb.SamplerError) as err:
        head.logits(x, a)
    assert err.value.code == -1
    other.logits(x, b)
    assert torch.equal(a, b)
    e.close()
    other.free()      # (the engine has freed it)


@pytest.mark.parametrize("rows,pad", [(2, 0), (16, 0), (70, 0), (70, 1), (140, 0)])
def test_captured_and_replayed(rows, pad):
    rng = np.random.default_rng(6)
    w, s, x = integers(rng, rows, 3000, 512 + 64 * pad, 64, "f16", "bf16")
    w, s, x = w[:, :256].contiguous(), s[:, :8].contiguous(), x[:, :512]     # (with a pad, rows off 16-byte boundaries)
    x = torch.nn.functional.pad(x, (0, pad))
    e = engine()
    head = e.load_head(w, s)
    outs = [torch.zeros(rows, 3000, device="cuda") for _ in range(2)]
    xs = [x.clone(), x.clone()]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs = []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        e.set_cuda_stream(streams[k].cuda_stream)
        with torch.cuda.graph(g, stream=streams[k]):
            head.logits(xs[k][:, :512], outs[k])
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(3):
        for k in range(2):
            xs[k][:, :512].copy_(torch.from_numpy(rng.integers(-7, 8, (rows, 512)).astype(np.float32)).cuda())
        torch.cuda.synchronize()
        for k in range(2):            # at the same time
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert torch.equal(outs[k].double(), plain(w, s, xs[k][:, :512]))
    e.close()


@pytest.mark.parametrize("rows,pad", [(3, 0), (16, 1), (40, 0), (40, 1), (140, 0)])
def test_queued_calls_read_their_own_hidden_states(rows, pad):
    """Calls queued one behind the other, hidden states that change between them, other work in front: each is placed while the one
    before it ends, and must not run ahead of it."""
    rng = np.random.default_rng(rows)
    w, s, _ = integers(rng, rows, 9000, 256, 32, "f16", "bf16")
    e = engine()
    head = e.load_head(w, s)
    xs = [torch.from_numpy(rng.integers(-7, 8, (rows, 256 + pad)).astype(np.float32)).to(torch.bfloat16).cuda() for _ in range(8)]
    big = torch.zeros(1 << 26, device="cuda")
    x, outs = torch.zeros_like(xs[0]), [torch.zeros(rows, 9000, device="cuda") for _ in range(8)]
    for k in range(8):
        big.add_(1.0)                     # what comes before takes its time
        x.copy_(xs[k])
        head.logits(x[:, :256], outs[k])
        if k % 2:
            head.logits(x[:, :256], outs[k])
    torch.cuda.synchronize()
    for k in range(8):
        assert torch.equal(outs[k].double(), plain(w, s, xs[k][:, :256])), k
    e.close()


def test_refusals():
    rng = np.random.default_rng(7)
    w, s, x = integers(rng, 2, 100, 128, 32, "f16", "bf16")
    e = engine()

    def code(f):
        with pytest.raises(fb.SamplerError) as err:
            f()
        return err.value.code

    assert code(lambda: e.load_head(w, torch.ones(100, 8, dtype=torch.float16, device="cuda"))) == -2          # groups of 16
    assert code(lambda: e.load_head(w[:, :56].contiguous(), torch.ones(100, 7, dtype=torch.float16, device="cuda"))) == -2
    assert code(lambda: e.load_head(torch.zeros(2, 16384 // 2 + 16, dtype=torch.uint8, device="cuda"), torch.ones(2, 513, dtype=torch.float16, device="cuda"))) == -2
    for bad in (lambda: e.load_head(w.int(), s), lambda: e.load_head(w, s.float())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: e.load_head(w[:, ::2], s), lambda: e.load_head(w[:50], s), lambda: e.load_head(w.cpu(), s),
                lambda: e.load_head(w, torch.ones(100, 3, dtype=torch.float16, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    head = e.load_head(w, s)
    out = torch.empty(2, 100, device="cuda")
    assert code(lambda: head.logits(x.float(), out)) == -1
    both = torch.zeros(4096, device="cuda")
    assert code(lambda: head.logits(both.view(torch.bfloat16)[:256].view(2, 128), both[:200].view(2, 100))) == -1
    for bad in (lambda: head.logits(x[:, :64], out), lambda: head.logits(x, out[:1]), lambda: head.logits(x, out.half()), lambda: head.logits(x.cpu(), out),
                lambda: head.logits(torch.zeros(128, 2, dtype=torch.bfloat16, device="cuda").T, out)):
        with pytest.raises(ValueError):
            bad()
    other = engine()
    with pytest.raises(ValueError):
        other.sample_hidden(head, [0], x[:1])
    L = e.lib
    assert L.fsb_head_logits(other._h, head._ptr, 2, x.data_ptr(), 1, 128, out.data_ptr(), 100) == -1
    assert L.fsb_head_logits(e._h, head._ptr, 0, x.data_ptr(), 1, 128, out.data_ptr(), 100) == -1
    assert L.fsb_head_logits(e._h, head._ptr, 65536, x.data_ptr(), 1, 128, out.data_ptr(), 100) == -3
    assert L.fsb_head_logits(e._h, head._ptr, 2, x.data_ptr() + 1, 1, 128, out.data_ptr(), 100) == -1
    assert L.fsb_head_logits(e._h, head._ptr, 2, x.data_ptr(), 1, 127, out.data_ptr(), 100) == -1
    assert L.fsb_head_logits(e._h, head._ptr, 2, x.data_ptr(), 1, 128, out.data_ptr(), 99) == -1
    assert L.fsb_head_logits(e._h, None, 2, x.data_ptr(), 1, 128, out.data_ptr(), 100) == -1
    assert L.fsb_head_free(other._h, head._ptr) == -1
    head.logits(x, out)
    assert torch.equal(out.double(), plain(w, s, x))
    other.close()
    e.close()
