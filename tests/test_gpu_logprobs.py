"""Token log probabilities, entropy and alternatives against 64 bits."""
import numpy as np
import pytest

import omnivoice_amd as ov

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def guided(c, u, g):
    """The float32 steps of the definition."""
    c = c.astype(np.float32)
    if u is None:
        return c.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        z = c + np.float32(g) * (c - u.astype(np.float32))
    return np.where(c == -np.inf, -np.inf, z).astype(np.float64)


def plain(z, tokens, top, mask):
    """(logprob, entropy, ids, their log probabilities) in 64 bits."""
    rows, vocab = z.shape
    ids = np.full((rows, top), -1)
    best = np.full((rows, top), -np.inf)
    logprob = np.full(rows, np.nan)
    entropy = np.full(rows, np.nan)
    for r in range(rows):
        m = z[r].max()
        if np.isnan(z[r]).any() or not np.isfinite(m):
            best[r] = np.nan
            continue
        d = z[r] - m
        e = np.exp(d)
        log_s = np.log(e.sum())
        logprob[r] = d[tokens[r]] - log_s if 0 <= tokens[r] < vocab else -np.inf
        entropy[r] = log_s - (e[e > 0] * d[e > 0]).sum() / e.sum()
        order = np.argsort(-z[r], kind="stable")[:top + 1]
        order = [i for i in order if i != mask and z[r, i] > -np.inf][:top]
        ids[r, :len(order)] = order
        best[r, :len(order)] = d[order] - log_s
    return logprob, entropy, ids, best


def call(c, u, tokens, top, g, mask, **more):
    rows = c.shape[0]
    out = [torch.full((rows,), 9.0, device="cuda"), torch.full((rows,), 9.0, device="cuda"),
           torch.full((rows, top), 9, dtype=torch.int32, device="cuda"),
           torch.full((rows, top), 9.0, device="cuda")]
    ov.op_token_logprobs(c, torch.tensor(np.asarray(tokens, np.int32)).cuda(), out[0], out[1],
                         out[2], out[3], uncond=u, guidance=g, mask_id=mask, **more)
    return out


def check(c, u, tokens, top, g, mask, **more):
    """Against 64 bits. A sum of n positive terms, n / 64 of them one after the
    other, is off by (n / 64 + 16) 2^-24 of itself and each term by as many
    halves of a step as its exponent's size, which the sum weighs by p: bounded by
    8 and by the entropy; the subtractions by one half step of what they give."""
    got = [x.cpu().numpy() for x in call(c, u, tokens, top, g, mask, **more)]
    z = guided(c.float().cpu().numpy(), None if u is None else u.float().cpu().numpy(), g)
    want = plain(z, tokens, top, mask)
    np.testing.assert_array_equal(got[2], want[2])
    h = np.nan_to_num(want[1], nan=0.0)
    base = (c.shape[1] / 64 + 32 + 4 * h) * 2.0 ** -24
    for k, grow in ((0, 1.0), (3, 1.0), (1, 1.0 + h)):
        finite = np.isfinite(want[k])
        np.testing.assert_array_equal(np.isnan(got[k]), np.isnan(want[k]))
        np.testing.assert_array_equal(got[k][~finite & ~np.isnan(want[k])],
                                      want[k][~finite & ~np.isnan(want[k])])
        tol = base * grow
        tol = tol[:, None] if k == 3 else tol
        err = np.abs(got[k].astype(np.float64) - want[k])
        tol = np.broadcast_to(tol + 4 * 2.0 ** -24 * np.abs(np.where(finite, want[k], 0.0)),
                              err.shape)
        assert (err[finite] <= tol[finite]).all(), (k, (err / tol)[finite].max())
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (3, 2, 5), (7, 63, 4), (5, 64, 32), (5, 65, 1), (40, 1025, 5), (9, 1024, 0),
    (3, 4095, 8), (2, 4097, 8), (3, 16385, 20), (2, 151936, 10), (1, 200001, 32), (300, 500, 3)])
def test_matches_plain(dtype, rows, vocab, top):
    rng = np.random.default_rng(rows + vocab)
    c = torch.from_numpy((rng.standard_normal((rows, vocab)) * 3).astype(np.float32)) \
        .to(TYPES[dtype]).cuda()
    tokens = rng.integers(0, vocab, rows)
    check(c, None, tokens, top, 0.0, None)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,top", [(50, 1025, 5), (3, 30001, 12), (9, 100, 32)])
@pytest.mark.parametrize("g", [2.0, 0.0, -0.7])
def test_guided_matches_plain(dtype, rows, vocab, top, g):
    rng = np.random.default_rng(vocab)
    c, u = (torch.from_numpy((rng.standard_normal((rows, vocab)) * 2).astype(np.float32))
            .to(TYPES[dtype]).cuda() for _ in range(2))
    check(c, u, rng.integers(0, vocab, rows), top, g, vocab - 1)


def test_first_alternative_is_what_score_predicts():
    """With the generator's sizes, guidance and mask: the best alternative and
    its log probability are op_score's prediction and confidence (its guided
    logits are normalised ones, two roundings apart)."""
    rng = np.random.default_rng(3)
    frames, codebooks, vocab = 50, 8, 1025
    logits = torch.from_numpy((rng.standard_normal((2 * frames, codebooks * vocab)) * 3)
                              .astype(np.float32)).cuda()
    prediction = torch.zeros(codebooks * frames, dtype=torch.int32, device="cuda")
    confidence = torch.zeros(codebooks * frames, device="cuda")
    ov.op_score(logits, prediction, confidence, frames, codebooks, vocab, vocab - 1, 2.0)
    c, u = logits[:frames].view(-1, vocab), logits[frames:].view(-1, vocab)
    out = call(c, u, np.zeros(frames * codebooks, np.int32), 2, 2.0, vocab - 1)
    ids = out[2].view(frames, codebooks, 2)[..., 0].t().reshape(-1)
    best = out[3].view(frames, codebooks, 2)
    near = (best[..., 0] - best[..., 1]).t().reshape(-1) < 1e-4  # a tie but for roundings
    assert torch.equal(ids[~near], prediction[~near]) and near.sum() < 10
    # z and log Z of magnitude 40, four roundings of 2^-24 each way.
    assert (best[..., 0].t().reshape(-1) - confidence).abs().max().item() < 40 * 8 * 2.0 ** -24


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("vocab", [20, 65, 98, 130, 500, 1024, 1040, 2500])
def test_long_lists_of_small_vocabularies(dtype, vocab):
    """More tokens listed than there are runs of 16, magnitudes far apart, both
    signs, and levels that more than 64 tokens share."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((7, vocab)).astype(np.float32)
    x[1] = 10.0 ** rng.uniform(-4, 3, vocab) * rng.choice([-1.0, 1.0], vocab)
    x[2] = -10.0 ** rng.uniform(-4, 3, vocab)
    x[3] = np.round(x[3])                            # a few levels
    x[4] = np.where(rng.random(vocab) < 0.7, 1.0, x[4])  # most of them one
    x[5] = np.where(rng.random(vocab) < 0.7, -np.inf, x[5])
    x[6] = np.where(np.arange(vocab) % 3 == 1, 0.0, -0.0)  # one value
    c = torch.from_numpy(x).to(TYPES[dtype]).cuda()
    for top, mask in ((1, None), (7, vocab // 2), (20, 0), (32, vocab - 1)):
        check(c, None, rng.integers(0, vocab, 7), top, 0.0, mask)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("vocab", [100, 1025, 5000, 70000])
def test_ties_go_to_the_lowest_index(dtype, vocab):
    rng = np.random.default_rng(4)
    rows = 6
    x = np.zeros((rows, vocab), np.float32)          # row 0: all equal
    x[1] = rng.integers(-2, 3, vocab)                # five values
    x[2, rng.permutation(vocab)[:40]] = 5.0          # forty best ones
    x[3] = -np.arange(vocab) // 64                   # falling in runs
    x[4] = np.arange(vocab) // 128                   # rising in runs
    x[5, -3:] = 1.0
    c = torch.from_numpy(x).to(TYPES[dtype]).cuda()
    for mask in (None, 0, int(np.argmax(x[2])), vocab - 1):
        check(c, None, rng.integers(0, vocab, rows), 32, 0.0, mask)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("step", [16, 1024, 4096, 8192, 1040])
@pytest.mark.parametrize("mask", [None, 80])
def test_best_tokens_in_a_row_of_steps(dtype, step, mask):
    """The best tokens every so many places apart, rising and falling, among
    smaller ones: all in one lane's runs, in one run, in one wave's, and equal."""
    rng = np.random.default_rng(step)
    vocab = 150000
    x = rng.random((3, vocab)).astype(np.float32)
    at = 80 + np.arange(36) * step
    at = at[at < vocab]
    x[0, at] = 5 + np.arange(len(at)) / 4
    x[1, at] = 50 - np.arange(len(at)) / 4
    x[2, at] = 7.0
    c = torch.from_numpy(x).to(TYPES[dtype]).cuda()
    got = check(c, None, [80, 81, 149999], 32, 0.0, mask)
    # The same rows many times: whole in a work-group each instead of split.
    many = call(c.repeat(200, 1), None, [80, 81, 149999] * 200, 7, 0.0, mask)
    np.testing.assert_array_equal(many[2].cpu().numpy(), np.tile(got[2][:, :7], (200, 1)))
    np.testing.assert_allclose(many[3].cpu().numpy(), np.tile(got[3][:, :7], (200, 1)),
                               atol=2 * (vocab / 64 + 40) * 2.0 ** -24)


@pytest.mark.parametrize("vocab", [70, 1025, 40000])
def test_infinities_nan_and_tokens_without_a_place(vocab):
    rng = np.random.default_rng(5)
    rows, inf = 12, np.inf
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    x[0] = -inf                                   # no distribution
    x[1, vocab // 2] = np.nan
    x[2, 3] = inf
    x[3] = -inf
    x[3, vocab - 1] = 7.0                         # one possible token
    x[4, rng.random(vocab) < 0.9] = -inf
    x[4, :3] = 0.0
    x[5] = 3e38                                   # large, all finite
    x[6] = -3e38
    x[7, ::2] = -1e30
    x[8, 5] = 1e4                                 # certain
    x[9, vocab - 1] = np.nan
    tokens = rng.integers(0, vocab, rows)
    tokens[3] = vocab - 1
    tokens[4] = int(np.argmin(x[4]))              # impossible
    tokens[10], tokens[11] = -1, vocab
    c = torch.from_numpy(x).cuda()
    got = check(c, None, tokens, 8, 0.0, None)
    assert got[0][4] == -inf and got[0][10] == -inf and got[0][11] == -inf
    assert (got[2][3] == [vocab - 1] + [-1] * 7).all()
    masked = check(c, None, tokens, 8, 0.0, vocab - 1)
    assert (masked[2][3] == -1).all() and (masked[3][3] == -inf).all()
    u = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32)).cuda()
    u[4] = c[4]                                   # impossible in both
    u[10, 0] = -inf                               # only there: no distribution
    check(c, u, tokens, 8, 2.0, None)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("offset,extra", [(0, 3), (1, 0), (3, 5), (8, 8)])
@pytest.mark.parametrize("vocab", [1025, 20000])
def test_rows_at_any_stride_and_alignment(dtype, offset, extra, vocab):
    """Rows inside wider ones whose neighbours are NaN: nothing past a row is
    taken into it."""
    rng = np.random.default_rng(6)
    rows = 9
    flat = torch.full((rows * (vocab + extra) + 32,), float("nan"), dtype=TYPES[dtype],
                      device="cuda")
    c = flat[offset:offset + rows * (vocab + extra)].view(rows, vocab + extra)[:, :vocab]
    c.copy_(torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32)))
    check(c, None, rng.integers(0, vocab, rows), 6, 0.0, None)
    check(c, torch.zeros_like(c), rng.integers(0, vocab, rows), 6, 1.0, None)


def test_what_is_not_asked_for():
    rng = np.random.default_rng(7)
    c = torch.from_numpy(rng.standard_normal((5, 3000)).astype(np.float32)).cuda()
    full = call(c, None, [1, 2, 3, 4, 5], 4, 0.0, None)
    entropy = torch.zeros(5, device="cuda")
    ov.op_token_logprobs(c, None, None, entropy)
    assert torch.equal(entropy, full[1])
    ids, best = torch.zeros_like(full[2]), torch.zeros_like(full[3])
    ov.op_token_logprobs(c, None, None, None, ids, best)
    assert torch.equal(ids, full[2]) and torch.equal(best, full[3])


def test_same_bits_every_time_and_in_a_graph():
    rng = np.random.default_rng(8)
    c = torch.from_numpy(rng.standard_normal((3, 90001)).astype(np.float32)).half().cuda()
    first = call(c, None, [1, 2, 3], 9, 0.0, None)
    again = call(c, None, [1, 2, 3], 9, 0.0, None)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    size = ov.lib().ovg_op_token_logprobs_workspace(3, 90001, 9)
    space = torch.full((size + 64,), 255, dtype=torch.uint8, device="cuda")
    tokens = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    out = [torch.zeros_like(x) for x in first]
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            ov.op_token_logprobs(c, tokens, *out, workspace=space[:size + 16])
    torch.cuda.current_stream().wait_stream(side)
    for k in range(3):
        for x in out:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, out)), k
        call(c, None, [4, 5, 6], 2, 0.0, None)
    assert (space[size + 16:] == 255).all()
    if size:
        with pytest.raises(ov.GeneratorError, match="^token logprobs: workspace"):
            ov.op_token_logprobs(c, tokens, *out, workspace=space[:size - 1])


def test_tensors_are_checked():
    c = torch.zeros((4, 30), device="cuda")
    i4, f4 = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    bad = [dict(tokens=i4.long()), dict(tokens=i4[:3]), dict(tokens=i4.cpu()),
           dict(logprob=f4.half()), dict(entropy=f4[:2]), dict(logits=c[0]),
           dict(logits=c.double()), dict(logits=c.t()), dict(uncond=c[:3]),
           dict(uncond=c.half()), dict(top_ids=torch.zeros((4, 2), dtype=torch.int32,
                                                           device="cuda")),
           dict(top_ids=torch.zeros((4, 33), dtype=torch.int32, device="cuda"),
                top_logprobs=torch.zeros((4, 33), device="cuda")),
           dict(logits=c.cpu(), tokens=i4.cpu(), logprob=f4.cpu(), entropy=f4.cpu())]
    for over in bad:
        args = dict(logits=c, tokens=i4, logprob=f4, entropy=f4.clone())
        args.update(over)
        with pytest.raises(ov.GeneratorError):
            ov.op_token_logprobs(**args)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("vocab", [40, 100, 1025, 2500, 40000, 151936])
def test_masks_of_the_types_lowest_value(dtype, vocab):
    """Masked ranges hold the type's lowest value, not -infinity: a lane's run, the
    elements before the first 16-byte border and behind the last, whole waves and
    whole splits; and the same from a logit next to the largest one. Few rows are
    split over work-groups, many are not."""
    rng = np.random.default_rng(vocab)
    low, high = (float(f(torch.finfo(TYPES[dtype]))) for f in
                 (lambda t: t.min, lambda t: t.max))
    x = rng.standard_normal((9, vocab)).astype(np.float32)
    x[0, 16:40] = low
    x[1, :17] = x[1, -17:] = low
    x[2, 5:] = low
    x[3, :vocab - 5] = low
    x[4, :vocab // 2] = low
    x[5, vocab // 2:] = low
    x[6, np.arange(vocab) // 1024 % 3 != 1] = low
    x[6, -1] = 0.0
    x[7, :vocab // 2] = low
    x[7, vocab // 2:] = high
    x[8, :vocab - 1] = low
    tokens = np.array([50 % vocab, 20, 2, vocab - 2, vocab - 1, 0, vocab - 1, vocab - 1, 0])
    flat = torch.empty((900, vocab + 3), dtype=TYPES[dtype], device="cuda")
    c = flat[:, 1:vocab + 1]
    c.copy_(torch.from_numpy(x).cuda().repeat(100, 1))
    got = check(c[:9], None, tokens, 5, 0.0, None)
    assert np.isfinite(got[1]).all()
    check(c[:9], None, tokens, 5, 0.0, vocab // 3)
    many = call(c, None, np.tile(tokens, 100), 5, 0.0, None)
    want = plain(c[:9].double().cpu().numpy(), tokens, 5, None)[1]
    # check()'s tolerance of the entropy.
    tol = (vocab / 64 + 32 + 4 * want) * 2.0 ** -24 * (1 + want) + 4 * 2.0 ** -24 * want
    err = np.abs(many[1].double().cpu().numpy().reshape(100, 9) - want)
    assert (err <= tol).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [100, 1025, 40000])
def test_guided_masks_far_below(dtype, vocab):
    """Masked logits whose guided ones are near float32's lowest, and masked in both."""
    rng = np.random.default_rng(vocab)
    c, u = rng.standard_normal((2, 4, vocab)).astype(np.float32)
    c[0, 16:60] = -1e38
    c[1, :vocab // 2] = -1e38
    c[2, 30:] = u[2, 30:] = float(torch.finfo(TYPES[dtype]).min)
    c[3, :vocab - 3] = -3e37
    c, u = (torch.from_numpy(x).to(TYPES[dtype]).cuda() for x in (c, u))
    got = check(c, u, [1, vocab - 1, 2, vocab - 2], 3, 2.0, None)
    assert np.isfinite(got[1]).all()


def test_rows_past_32_bits():
    """Rows more than 2^31 elements apart, conditional and unconditional."""
    rng = np.random.default_rng(9)
    vocab = 1025
    flat = torch.empty((2 << 31) + (1 << 16), dtype=torch.float16, device="cuda")
    c, u = (flat[at:].as_strided((3, vocab), (1 << 31, 1)) for at in (0, 1 << 12))
    for x in (c, u):
        x.copy_(torch.from_numpy(rng.standard_normal((3, vocab)).astype(np.float32)))
    check(c, None, [5, 0, 1024], 6, 0.0, None)
    check(c, u, [5, 0, 1024], 6, 2.0, 1024)
