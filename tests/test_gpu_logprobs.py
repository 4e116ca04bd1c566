"""TokenLogprobs against its 64-bit restatement.

ids are a function of the logits' order and compared exactly. Numbers, from
the arithmetic: the sum of V exponentials (each within 2^-21 of itself with
its argument's rounding, at most 100 2^-24) is off by at most (2^-17 + V_eff
2^-23) of itself with V_eff = 64 additions in a row on a tree of partial sums;
ln of it is off by as much, and x - m and the final difference by 2^-24 each
of their size."""
import math

import numpy as np
import pytest

from oracle import kv_quant_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env(cuda):
    from orator_b200 import ops
    return cuda, ops


def score(env, x, targets, top, stride=None, stream=None, parts=(True, True)):
    """x [rows, vocab] on the GPU, rows `stride` apart."""
    torch, ops = env
    rows, vocab = x.shape
    lp, ent = torch.full((rows + 1,), 7.0, device="cuda"), torch.full((rows + 1,), 7.0, device="cuda")
    ids = torch.full((rows + 1, max(top, 1)), -7, dtype=torch.int32, device="cuda")
    tl = torch.full((rows + 1, max(top, 1)), 7.0, device="cuda")
    ops.TokenLogprobs(x.data_ptr(), 0 if x.dtype == torch.float32 else 1, rows, vocab, x.stride(0) if rows > 1 else max(vocab, x.stride(0)),
                      targets.data_ptr() if parts[0] else 0, top, lp.data_ptr() if parts[0] else 0, ent.data_ptr() if parts[1] else 0,
                      ids.data_ptr() if top else 0, tl.data_ptr() if top else 0, stream)
    torch.cuda.synchronize()
    assert lp[rows] == 7 and ent[rows] == 7 and (ids[rows] == -7).all() and (tl[rows] == 7).all()
    return lp[:rows].cpu().numpy(), ent[:rows].cpu().numpy(), ids[:rows].cpu().numpy(), tl[:rows].cpu().numpy()


def check(env, x, targets, top, got):
    lp, ent, ids, tl = O.token_scores(x.double().cpu().numpy(), targets.cpu().numpy(), top)
    finite = x.double().cpu().numpy()
    size = np.abs(np.where(np.isfinite(finite), finite, 0)).max(1)
    bar = 2.0**-17 + 64 * 2.0**-23 + 2.0**-22 * size
    for a, b in ((got[0], lp), (got[3], tl)):
        bars = bar if b.ndim == 1 else np.broadcast_to(bar[:, None], b.shape)
        if b.size == 0 or (b.ndim == 2 and top == 0):
            continue
        inf = np.isneginf(b)
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(np.isneginf(a), inf)
        with np.errstate(invalid="ignore"):
            assert (np.abs(a - b)[np.isfinite(b)] <= bars[np.isfinite(b)]).all(), np.nanmax(np.abs(a - b)[np.isfinite(b)])
    assert np.array_equal(np.isnan(got[1]), np.isnan(ent))
    fine = ~np.isnan(ent)
    # entropy: ln l as above, and the sum of (x - m) e^(x - m), each term off by 2^-17 of itself as well
    assert (np.abs(got[1] - ent)[fine] <= bar[fine] * (1 + 2 * ent[fine])).all()
    if top:
        assert np.array_equal(got[2], ids)


SHAPES = [(1, 1, 1), (3, 2, 2), (2, 31, 5), (5, 33, 32), (4, 1000, 7), (1, 4097, 20), (3, 65537, 32), (2, 151936, 5), (70, 5000, 1),
          (9, 10241, 0), (300, 129, 3), (1, 300001, 10),
          (5, 1000, 32), (3, 4999, 32), (2, 9001, 31)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab,top", SHAPES)
def test_scores(env, dtype, rows, vocab, top):
    torch, _ = env
    g = torch.Generator().manual_seed(rows + vocab)
    x = (3 * torch.randn(rows, vocab + 3, generator=g)).to(getattr(torch, dtype)).cuda()[:, :vocab]  # rows of odd stride: ties in bf16
    t = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32)
    t[::3] = -1
    t[1::5] = vocab
    t = t.cuda()
    got = score(env, x, t, top)
    check(env, x, t, top, got)
    assert all(np.array_equal(a, b) for a, b in zip(got, score(env, x, t, top)))
    assert (got[0][t.cpu().numpy() < 0] == 0).all() and (got[0][t.cpu().numpy() >= vocab] == 0).all()
    # every part alone gives the same numbers
    assert np.array_equal(score(env, x, t, top, parts=(False, True))[1], got[1])
    assert np.array_equal(score(env, x, t, 0, parts=(True, False))[0], got[0])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [33, 5000, 40000])
def test_orders(env, dtype, vocab):
    """Logits whose order is what a selection finds hard: equal, rising, falling, the largest side by side, two values, -inf."""
    torch, _ = env
    i = torch.arange(vocab, dtype=torch.float32)
    rows = [torch.zeros(vocab), i / vocab, -i / vocab, torch.where(i < 200, 5 + i / 1000, -i / vocab), (i % 2),
            torch.where(i == vocab - 1, 3.0, -math.inf), torch.where(i < 3, 1.0, -math.inf), -torch.zeros(vocab) + torch.where(i % 3 == 0, -0.0, 0.0),
            torch.where(i >= vocab - 20, 1.0, 0.0), torch.full((vocab,), -3e38), torch.where(i == 7, 1e30, -1e30)]
    x = torch.stack(rows).to(getattr(torch, dtype)).cuda()
    t = torch.full((len(rows),), 7, dtype=torch.int32, device="cuda")
    check(env, x, t, 32, score(env, x, t, 32))


@pytest.mark.parametrize("vocab", [40, 30000])
def test_rows_without_distribution(env, vocab):
    """NaN, +inf and rows of -inf: NaN numbers, ids that rank what there is; the other rows are untouched."""
    torch, _ = env
    x = torch.randn(6, vocab, generator=torch.Generator().manual_seed(0))
    x[1, 5] = math.nan
    x[2, 3] = math.inf
    x[3] = -math.inf
    x[4] = math.nan
    x = x.cuda()
    t = torch.zeros(6, dtype=torch.int32, device="cuda")
    got = score(env, x, t, 10)
    check(env, x, t, 10, got)
    assert np.isnan(got[0]).tolist() == [False, True, True, True, True, False]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 40, 5), (1, 5000, 32), (1, 151936, 5), (700, 9001, 20)])
def test_nan_beside_other_logits(env, dtype, rows, vocab, top):
    """A NaN anywhere, whatever its neighbours and the logits behind it are: NaN numbers, and ids that rank every other logit."""
    torch, _ = env
    i = torch.arange(vocab)
    some = torch.randn(vocab, generator=torch.Generator().manual_seed(vocab))
    lowest = torch.finfo(getattr(torch, dtype)).min
    for at in (0, 5, vocab // 2, vocab - 1):
        one = []
        for rest in (some, torch.where(i == vocab // 3, 1.0, -math.inf), torch.full((vocab,), -math.inf), torch.where(i < 30, 2.0, lowest)):
            x = rest.clone()
            x[at] = math.nan
            for k in range(1, 4):  # the largest in the same 16 bytes and far away
                x[(at + k) % vocab], x[(at + 17 * k * k) % vocab] = 40.0 + k, 50.0 - k
            one += [x, rest.clone()]
            one[-1][at] = math.nan
        x = torch.stack(one).to(getattr(torch, dtype))
        x = x[torch.arange(rows) % len(one)] if rows > 1 else x
        t = torch.full((len(x),), vocab // 3, dtype=torch.int32, device="cuda")
        for part in [x] if rows > 1 else x[:, None]:
            part = part.cuda()
            got = score(env, part, t[:len(part)], top)
            check(env, part[:8], t[:min(8, len(part))], top, [g[:8] for g in got])
            assert np.isnan(got[0]).all() and np.isnan(got[1]).all() and np.isnan(got[3]).all()
            assert all(np.array_equal(g[k], g[k % 8], equal_nan=True) for g in got for k in range(8, len(part)))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [100, 5000, 40000])
def test_masks_of_the_lowest_value(env, dtype, vocab):
    """A row masked with its type's lowest value is the row masked with -inf, wherever the mask lies: both have weight 0."""
    torch, _ = env
    i = torch.arange(vocab)
    keep = torch.stack([i >= vocab // 2, i < vocab // 2, i >= vocab - 40, i < 40, i % (vocab // 33) == 0, (i >= vocab // 3) & (i < vocab // 3 + 35)])
    x = (5 * torch.randn(len(keep), vocab, generator=torch.Generator().manual_seed(vocab))).to(getattr(torch, dtype))
    t = keep.int().argmax(1).int().cuda()
    lowest = torch.where(keep, x, torch.finfo(x.dtype).min).cuda()
    none = torch.where(keep, x, -math.inf).to(x.dtype).cuda()
    got, want = score(env, lowest, t, 32), score(env, none, t, 32)
    check(env, none, t, 32, want)
    assert all(np.array_equal(a, b) for a, b in zip(got, want))
    masked = (~keep).int().argmax(1).int().cuda()
    lp = score(env, lowest, masked, 1)[0]
    assert (np.abs(lp / torch.finfo(x.dtype).min - 1) <= 2.0**-20).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 700, 32), (1, 5000, 5), (1, 30000, 32), (1, 151936, 20), (1, 1 << 19, 32), (600, 40000, 32), (300, 151936, 5)])
def test_few_legal_tokens(env, dtype, rows, vocab, top):
    """Rows masked down to some tokens, with -inf or the type's lowest value: the places behind them go to the lowest masked ids."""
    torch, _ = env
    tt = getattr(torch, dtype)
    i = torch.arange(vocab)
    g = torch.Generator().manual_seed(vocab + top)
    at = torch.randperm(vocab, generator=g)
    per = 8 if dtype == "bfloat16" else 4  # values of 16 bytes
    keeps = [i < 3, i >= vocab - 3, torch.isin(i, at[:3]), torch.isin(i, at[:100]), (i >= vocab // 2) & (i < vocab // 2 + 1000),
             i % (32 * per) < 8 * per,     # every batch, but a quarter of its lanes
             i // (128 * per) % 9 == 3, i < 0, i >= 0,
             (i // (128 * per) == 2) & (i // per % 32 < 31)]  # all values of 31 lanes
    vals = [2 * torch.randn(vocab, generator=g), torch.randint(0, 3, (vocab,), generator=g).float(), torch.zeros(vocab)]
    x = torch.stack([torch.where(k, v, mask) for k in keeps for v in vals for mask in (-math.inf, torch.finfo(tt).min)]).to(tt)
    t = torch.stack([at[0], at[1]] * (len(x) // 2)).int().cuda()
    if rows == 1:
        for r in range(len(x)):
            part = x[r:r + 1].cuda()
            check(env, part, t[r:r + 1], top, score(env, part, t[r:r + 1], top))
        return
    pick = torch.arange(rows) % len(x)
    part, want = x[pick].cuda(), t[pick.cuda()]
    got = score(env, part, want, top)
    check(env, part[:len(x)], t, top, [a[:len(x)] for a in got])
    assert all(np.array_equal(a[r], a[r % len(x)], equal_nan=True) for a in got for r in range(len(x), rows))


def test_sure_rows(env):
    """Entropies far below one keep their digits."""
    torch, _ = env
    x = torch.full((4, 20000), -1.0)
    for r, gap in enumerate((12.0, 25.0, 40.0, 80.0)):
        x[r, 11] = gap
    x = x.cuda()
    t = torch.full((4,), 11, dtype=torch.int32, device="cuda")
    lp, ent, ids, _ = score(env, x, t, 1)
    want = O.token_scores(x.double().cpu().numpy(), t.cpu().numpy(), 1)
    assert (ids == 11).all()
    # relative: the exponential's argument is off by 2^-24 of at most 81, and the sums by less than 2^-17
    assert (np.abs(ent - want[1]) <= (81 * 2.0**-23 + 2.0**-16) * want[1]).all()
    assert (np.abs(lp - want[0]) <= (81 * 2.0**-23 + 2.0**-16) * np.abs(want[0])).all()


def test_far_rows(env):
    """Rows more than 2^31 elements apart."""
    torch, ops = env
    stride, vocab = (1 << 31) + 10, 2000
    buf = torch.empty(2 * stride + vocab, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(buf, (3, vocab), (stride, 1))
    x.copy_(torch.randn(3, vocab, generator=torch.Generator().manual_seed(0)))
    t = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    check(env, x, t, 4, score(env, x, t, 4))


def test_graph_and_streams(env):
    torch, ops = env
    x = torch.randn(8, 50000, generator=torch.Generator().manual_seed(0)).cuda()
    t = torch.arange(8, dtype=torch.int32, device="cuda")
    lp, ent = torch.empty(8, device="cuda"), torch.empty(8, device="cuda")
    ids, tl = torch.empty(8, 4, dtype=torch.int32, device="cuda"), torch.empty(8, 4, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.TokenLogprobs(x.data_ptr(), 0, 8, 50000, 50000, t.data_ptr(), 4, lp.data_ptr(), ent.data_ptr(), ids.data_ptr(), tl.data_ptr(),
                          torch.cuda.current_stream().cuda_stream)
    for seed in (1, 2):
        x.copy_(torch.randn(8, 50000, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = lp.cpu().numpy(), ent.cpu().numpy(), ids.cpu().numpy(), tl.cpu().numpy()
        check(env, x, t, 4, got)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        assert all(np.array_equal(a, b) for a, b in zip(got, score(env, x, t, 4, stream=s)))


def test_decoder_logits(env):
    """The decoder's own logits after a prefill: the greedy token's log probability, and the alternatives behind it."""
    torch, ops = env
    import ctypes as C
    from orator_b200 import AsrTextConfig, AsrTextDecoder, _lib
    from oracle import synth
    vocab = 4096
    dec = AsrTextDecoder(AsrTextConfig(num_layers=2, vocab_size=vocab, max_seq_len=64))
    dec.init_synthetic(7)
    dec.Prefill(synth.audio_rows(7, 12, 2048))
    p = C.c_void_p()
    _lib.call("orx_decoder_logits_device", dec._h, C.byref(p))
    host = torch.from_numpy(np.array(dec.CopyLogits(), np.float32))[None]
    best = dec.Argmax()
    t = torch.tensor([best], dtype=torch.int32, device="cuda")
    lp, ent = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
    ids, tl = torch.empty(1, 5, dtype=torch.int32, device="cuda"), torch.empty(1, 5, device="cuda")
    ops.TokenLogprobs(p.value, 0, 1, vocab, vocab, t.data_ptr(), 5, lp.data_ptr(), ent.data_ptr(), ids.data_ptr(), tl.data_ptr())
    torch.cuda.synchronize()
    check(env, host, t, 5, (lp.cpu().numpy(), ent.cpu().numpy(), ids.cpu().numpy(), tl.cpu().numpy()))
    assert ids[0, 0].item() == best and lp[0].item() == tl[0, 0].item()
    dec.close()
