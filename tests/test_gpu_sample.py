"""The draw of tokens against the definition in 64 bits."""
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
        return c
    with np.errstate(invalid="ignore", over="ignore"):
        z = c + np.float32(g) * (c - u.astype(np.float32))
    return np.where(c == -np.inf, np.float32(-np.inf), z).astype(np.float32)


def plain(z, u, temperature, top_k, top_p, min_p, mask):
    """A row's token, from the definition; a draw or a share's border would have to lie
    within 2^-40 of a token's for the two to differ."""
    z = z.astype(np.float64).copy()
    if mask is not None and 0 <= mask < len(z):
        z[mask] = -np.inf
    if np.isnan(z).any() or z.max() == np.inf or z.max() == -np.inf:
        return -1
    order = np.argsort(-z, kind="stable")
    if not temperature > 0:
        return int(order[0])
    order = order[z[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    w = np.exp((z[order] - z[order[0]]) / np.float64(np.float32(temperature)))
    w[w < 2.0 ** -50] = 0.0
    keep = np.ones(len(w), bool)
    if np.float32(top_p) < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        keep &= before < np.float64(np.float32(top_p)) * w.sum()
    keep &= w >= min(np.float64(np.float32(min_p)), 1.0)
    keep[0] = True
    kept = np.zeros(len(z))
    kept[order[keep]] = w[keep]
    total = np.cumsum(kept)
    u = min(max(float(u), 0.0), 1.0 - 2.0 ** -53)
    return int(np.argmax(total > u * total[-1]))


def each(value, rows):
    return value.tolist() if isinstance(value, torch.Tensor) else [value] * rows


def check(c, random, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=None, g=0.0, mask=None,
          extra=0):
    rows, vocab = c.shape

    def place(t):
        wide = torch.full((rows, vocab + extra), 50.0, dtype=t.dtype)
        wide[:, :vocab] = t
        return wide.cuda()[:, :vocab]

    def dev(v):
        return v.cuda() if isinstance(v, torch.Tensor) else v
    tokens = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    ov.op_sample(place(c), random.cuda(), tokens, dev(temperature), dev(top_k), dev(top_p),
                 dev(min_p), uncond=None if u is None else place(u), guidance=g, mask_id=mask)
    got = tokens.cpu().numpy()
    z = guided(c.float().numpy(), None if u is None else u.float().numpy(), g)
    want = [plain(z[r], random[r], t, k, p, m, mask) for r, (t, k, p, m) in
            enumerate(zip(*(each(v, rows) for v in (temperature, top_k, top_p, min_p))))]
    np.testing.assert_array_equal(got, want)
    return got


def logits_of(seed, rows, vocab, kind="f32", peaks=True):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, vocab, generator=g) * 2
    if peaks:
        z.scatter_add_(1, torch.randint(0, vocab, (rows, 6), generator=g),
                       torch.randn(rows, 6, generator=g) * 2 + 8)
    return z.to(TYPES[kind]), torch.rand(rows, generator=g)


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=50), dict(top_k=1),
            dict(top_p=0.9), dict(top_p=0.3, temperature=1.5), dict(min_p=0.05),
            dict(top_k=20, top_p=0.8, min_p=0.02, temperature=0.9), dict(top_k=100000),
            dict(temperature=20.0), dict(temperature=0.01), dict(top_k=500, top_p=0.99)]


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("rows,vocab,kind", [(1, 1, "f32"), (3, 2, "f16"), (40, 63, "bf16"),
                                             (30, 64, "f32"), (50, 1000, "f16"),
                                             (60, 1025, "f32"), (20, 2048, "bf16"),
                                             (9, 2049, "f32"), (7, 5003, "bf16"),
                                             (5, 20011, "f32"), (4, 65537, "f16"),
                                             (3, 151936, "bf16"), (2, 200003, "f32")])
def test_sample(settings, rows, vocab, kind):
    c, random = logits_of(vocab, rows, vocab, kind)
    check(c, random, extra=vocab % 3, **settings)


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("rows,vocab,kind", [(40, 100, "f16"), (60, 1025, "f32"),
                                             (10, 3000, "bf16"), (3, 50000, "f32")])
def test_guided_and_masked(settings, rows, vocab, kind):
    c, random = logits_of(1, rows, vocab, kind)
    u, _ = logits_of(2, rows, vocab, kind, peaks=False)
    check(c, random, u=u, g=2.0, mask=vocab - 1, **settings)
    top = int(c[0].float().argmax())
    check(c, random, mask=top, **settings)


@pytest.mark.parametrize("rows,vocab,kind", [(64, 500, "f32"), (64, 1025, "bf16"),
                                             (40, 9001, "f16"), (16, 151936, "bf16")])
def test_settings_of_each_row(rows, vocab, kind):
    c, random = logits_of(3, rows, vocab, kind)
    g = torch.Generator().manual_seed(4)

    def pick(values, dtype):
        return torch.tensor(values, dtype=dtype)[torch.randint(0, len(values), (rows,),
                                                               generator=g)]
    check(c, random, pick([0.0, 0.5, 1.0, 3.0, -1.0], torch.float32),
          pick([0, 1, 5, 100, 7000, -3], torch.int32),
          pick([1.0, 0.95, 0.5, 0.0, 2.0], torch.float32),
          pick([0.0, 0.01, 0.3, 1.0, 5.0, -1.0], torch.float32))


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("vocab", [7, 64, 1000, 1025, 2500, 30000])
def test_equal_logits(settings, vocab):
    """Few different values: thresholds fall among equals, which go by index. All equal:
    shares of whole numbers, whose borders are exact."""
    c = torch.randint(0, 4, (30, vocab), generator=torch.Generator().manual_seed(vocab)).float()
    random = torch.rand(30, generator=torch.Generator().manual_seed(5))
    check(c, random, **settings)
    check(torch.full((30, vocab), -3.0), random, **settings)
    signed = torch.where(c > 1, 0.0, -0.0)  # both zeros are one value
    check(signed, random, **settings)


@pytest.mark.parametrize("vocab", [5, 1024, 4096])
def test_a_half_share_of_equals(vocab):
    """top_p of 0.5 over an even number of equals keeps exactly half of them."""
    random = torch.linspace(0, 1, 40)[:-1].contiguous()
    got = check(torch.zeros(39, vocab).half(), random, top_p=0.5)
    # random numbers to 38 / 39 of the first (vocab + 1) // 2 tokens
    assert got.max() == (vocab + 1) // 2 * 38 // 39


@pytest.mark.parametrize("vocab", [3, 100, 1025, 3000, 40000])
def test_rows_without_numbers(vocab):
    c, random = logits_of(6, 12, vocab)
    c[1, vocab // 2] = np.nan
    c[2, 1] = np.inf
    c[3] = -np.inf
    c[4] = -np.inf
    c[4, vocab - 2] = -3.0
    c[5, ::2] = -np.inf
    c[6] = -np.inf
    c[6, 0] = 2.0
    c[7, 0] = np.nan
    c[8] = -3.4028234e38
    c[9, 1] = 3.4028234e38
    c[10, 1], c[10, 0] = 3.4028234e38, -3.4028234e38
    for settings in SETTINGS:
        got = check(c, random, mask=0, **settings)
        assert got[6] == -1 and got[1] == -1  # its only token is the mask's
        check(c, random, **settings)
    u = torch.zeros_like(c)
    u[11, 2] = -np.inf  # +inf
    u[0, 1] = np.nan
    check(c, random, u=u, g=1.5)
    check(c, random, u=u, g=0.0, top_k=3)


@pytest.mark.parametrize("vocab", [10, 1025, 9000])
def test_random_numbers_at_the_ends(vocab):
    c, _ = logits_of(7, 6, vocab)
    random = torch.tensor([0.0, 1.0 - 2.0 ** -24, 2.0 ** -30, 0.5, 1e-45, 0.25])
    for settings in SETTINGS:
        check(c, random, **settings)
    outside = torch.tensor([-1.0, 1.0, 7.0, -np.inf, np.inf, np.nan])
    tokens = torch.zeros(6, dtype=torch.int32, device="cuda")
    ov.op_sample(c.cuda(), outside.cuda(), tokens)
    got = tokens.cpu().numpy()
    assert got[5] == -1 and got[0] == 0 and got[3] == 0
    last = [plain(c[r].numpy(), 1 - 2.0 ** -24, 1.0, 0, 1.0, 0.0, None) for r in range(5)]
    assert all(got[r] >= last[r] for r in (1, 2, 4)) and got.max() < vocab


def test_numbers_that_are_none():
    c, random = logits_of(8, 4, 300)
    bad = torch.tensor([1.0, np.nan, 1.0, 0.5])
    for name in ("temperature", "top_p", "min_p"):
        tokens = torch.zeros(4, dtype=torch.int32, device="cuda")
        ov.op_sample(c.cuda(), random.cuda(), tokens, **{name: bad.cuda()})
        assert tokens[1] == -1 and (tokens[[0, 2, 3]] >= 0).all()
    check(c, random, temperature=torch.tensor([1e-45, 1e38, 1e-30, 3e38]))
    # At an infinite temperature all that can be drawn weigh the same.
    c[:, 100:] = -np.inf
    tokens = torch.zeros(4, dtype=torch.int32, device="cuda")
    ov.op_sample(c.cuda(), random.cuda(), tokens, temperature=float("inf"))
    np.testing.assert_array_equal(tokens.cpu(), np.floor(random.numpy().astype(np.float64) * 100))


@pytest.mark.parametrize("vocab", [7, 1500, 30000])
@pytest.mark.parametrize("min_p", [1.0, 1.5, np.inf])
def test_min_p_from_one_on(vocab, min_p):
    """The best and its equals, whichever of them is first."""
    c = torch.zeros(6, vocab)
    c[:, [1, vocab // 2, vocab - 1]] = 3.0
    got = check(c, torch.tensor([0.0, 0.3, 0.4, 0.6, 0.7, 0.99]), min_p=min_p)
    assert got.tolist() == [1, 1, vocab // 2, vocab // 2, vocab - 1, vocab - 1]


def test_no_rows_and_one_draw_many_times():
    tokens = torch.zeros(0, dtype=torch.int32, device="cuda")
    ov.op_sample(torch.zeros(0, 50, device="cuda"), torch.zeros(0, device="cuda"), tokens)
    c, _ = logits_of(9, 1, 151936, "bf16")
    rows = c.expand(200, -1).contiguous()
    random = torch.linspace(0, 1, 201)[:-1].contiguous()
    got = check(rows, random, top_k=30)
    assert (np.diff(got) >= 0).all()  # by index, as the random number grows


def test_rows_past_32_bit_offsets():
    rows, vocab = 16500, 131072
    c = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    c[torch.arange(rows), torch.arange(rows) * 7 % vocab] = 30.0
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    ov.op_sample(c, torch.rand(rows, device="cuda"), tokens, top_k=1)
    assert torch.equal(tokens.cpu().long(), torch.arange(rows) * 7 % vocab)


LONG = [dict(), dict(top_p=0.9), dict(top_k=40), dict(top_k=2000), dict(top_k=9000, top_p=0.95),
        dict(min_p=0.1), dict(top_p=0.999, min_p=0.3), dict(top_k=3000, min_p=0.5),
        dict(top_k=300, top_p=0.5, temperature=2.0), dict(temperature=3.0, top_p=0.99)]


@pytest.mark.parametrize("settings", LONG)
@pytest.mark.parametrize("rows,vocab,kind", [(3, 151936, "f32"), (2, 1100001, "bf16"),
                                             (1, 4300000, "f32")])
def test_many_kept_and_long_rows(settings, rows, vocab, kind):
    """Thresholds far down a row, a min_p above the one that top_p would set, rows of more
    parts than a work-group holds."""
    c, random = logits_of(vocab + 1, rows, vocab, kind)
    check(c, random, **settings)


@pytest.mark.parametrize("settings", [dict(), dict(top_k=300), dict(top_p=0.9), dict(top_k=30),
                                      dict(min_p=0.01)])
def test_more_rows_than_hold_a_state(settings):
    c, random = logits_of(11, 1100, 2600, "f16")
    check(c, random, **settings)


def test_settings_of_many_rows():
    rows = 700
    c, random = logits_of(12, rows, 4100, "bf16")
    g = torch.Generator().manual_seed(13)

    def pick(values, dtype):
        return torch.tensor(values, dtype=dtype)[torch.randint(0, len(values), (rows,),
                                                               generator=g)]
    check(c, random, pick([0.0, 0.6, 1.0, 2.0], torch.float32),
          pick([0, 3, 600, 5000], torch.int32), pick([1.0, 0.9, 0.4], torch.float32),
          pick([0.0, 0.05], torch.float32))


@pytest.mark.parametrize("top_k", [0, 10, 700, 3000])
def test_more_equals_than_a_list_holds(top_k):
    """Thousands of equal logits around the threshold, some above and below, in 8 rows."""
    c = torch.zeros(8, 40000)
    c[:, ::7] = 1.0
    c[:, 5::9] = -4.0
    c[1:, 100] = 9.0
    c[2, :] = 0.5
    random = torch.linspace(0, 1, 9)[:-1].contiguous()
    check(c, random, top_k=top_k)
    check(c, random, top_k=top_k, temperature=0.5, min_p=0.2)
    # Shares that end inside the equals, away from a token's border.
    check(c[:2], random[:2], top_k=top_k, top_p=0.61803)


def few_allowed(rows, vocab, allowed, values, seed=40):
    """Rows of -infinities with `allowed` tokens of so many different values, far enough
    apart in the row to lie in every part of it; 0: any values."""
    g = torch.Generator().manual_seed(seed)
    c = torch.full((rows, vocab), -np.inf)
    for r in range(rows):
        at = torch.randperm(vocab, generator=g)[:allowed]
        c[r, at] = -torch.randint(0, values, (allowed,), generator=g).float() if values else \
            torch.randn(allowed, generator=g)
    return c, torch.rand(rows, generator=g)


@pytest.mark.parametrize("values", [1, 2, 5, 0])
@pytest.mark.parametrize("vocab,allowed", [(20000, 3000), (20000, 6000), (151936, 3000)])
def test_fewer_tokens_than_top_k(vocab, allowed, values):
    """A top_k that all of the tokens fit into cuts nothing off: shares are of all of them,
    the last ones and their equals too. 3000 equal tokens with a share of 0.9: 2700."""
    c, random = few_allowed(6, vocab, allowed, values)
    for top_k in (allowed + 1, 9000):
        for settings in (dict(top_p=0.9), dict(top_p=0.95), dict(top_p=0.95, min_p=0.001),
                         dict(), dict(top_p=0.9, temperature=1e30), dict(temperature=3e38)):
            check(c, random, top_k=top_k, **settings)
    each_k = torch.tensor([allowed - 1, allowed, allowed + 1, 19999, 0, 5], dtype=torch.int32)
    check(c, random, top_k=each_k, top_p=torch.tensor([0.9, 1.0, 0.9, 0.97, 0.9, 0.8]))


LONG_ROW = 4300000  # more parts than a work-group holds in LDS


def test_long_rows_with_few_tokens():
    c, random = few_allowed(2, LONG_ROW, 10, 0)
    for settings in (dict(top_k=50), dict(top_k=9), dict(top_k=50, top_p=0.9),
                     dict(top_k=11, min_p=0.1)):
        check(c, random, **settings)


@pytest.mark.parametrize("settings", [dict(top_k=50, temperature=0.2),
                                      dict(top_k=2000, temperature=0.05),
                                      dict(top_k=3000, temperature=0.01, top_p=0.999)])
def test_long_rows_of_few_that_weigh(settings):
    """Fewer than top_k tokens weigh 2^-50 of the best."""
    c, random = logits_of(41, 2, LONG_ROW)
    check(c, random, **settings)


def test_long_rows_of_a_share_past_the_sums():
    """A best token, a share of nearly all, and millions that weigh less than a unit of the
    sums does: together 2^-19 of the row, whose parts the sums do not see."""
    c = torch.full((3, LONG_ROW), -28.5)
    c[:, 2000001] = 0.0
    check(c, torch.tensor([0.3, 0.5, 0.7]), top_p=1.0 - 2.0 ** -24)


def test_the_callers_workspace():
    """Nothing behind it is written, what is in it does not matter."""
    c, random = logits_of(14, 6, 30000, "bf16")
    need = ov.op_sample_workspace(6, 30000)
    for fill in (0, 255):
        space = torch.full((need + 4096,), fill, dtype=torch.uint8, device="cuda")
        for settings in (dict(), dict(top_k=20), dict(top_p=0.9), dict(top_k=900, min_p=0.01)):
            want = check(c, random, **settings)
            tokens = torch.zeros(6, dtype=torch.int32, device="cuda")
            ov.op_sample(c.cuda(), random.cuda(), tokens, workspace=space[:need], **settings)
            np.testing.assert_array_equal(tokens.cpu(), want)
        assert (space[need:] == fill).all()
    with pytest.raises(ov.GeneratorError, match="workspace"):
        ov.op_sample(c.cuda(), random.cuda(), tokens, workspace=space[:need - 16])


def test_two_captured_draws_at_once():
    """Two graphs with workspaces of their own, replayed on two streams at once, with eager
    draws between; each follows its logits."""
    rows, vocab = 40, 30000
    settings = [dict(top_p=0.9, temperature=0.8), dict(top_k=700, min_p=0.001)]
    draws = []
    for i, s in enumerate(settings):
        d = dict(c=torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda"),
                 random=torch.zeros(rows, device="cuda"),
                 tokens=torch.zeros(rows, dtype=torch.int32, device="cuda"),
                 space=torch.zeros(ov.op_sample_workspace(rows, vocab), dtype=torch.uint8,
                                   device="cuda"),
                 stream=torch.cuda.Stream(), graph=torch.cuda.CUDAGraph())
        torch.cuda.synchronize()
        with torch.cuda.graph(d["graph"], stream=d["stream"]):
            ov.op_sample(d["c"], d["random"], d["tokens"], workspace=d["space"], **s)
        draws.append(d)
    for t in range(4):
        inputs = [logits_of(20 + 2 * t + i, rows, vocab, "bf16") for i in range(2)]
        for d, (c, random) in zip(draws, inputs):
            d["c"].copy_(c)
            d["random"].copy_(random)
            d["tokens"].fill_(-9)
        torch.cuda.synchronize()
        for d in draws:
            with torch.cuda.stream(d["stream"]):
                d["graph"].replay()
        want = [check(c, random, **s) for (c, random), s in zip(inputs, settings)]
        torch.cuda.synchronize()
        for d, w in zip(draws, want):
            np.testing.assert_array_equal(d["tokens"].cpu(), w)


def test_threads():
    """Calls of several host threads, each on a stream of its own."""
    import threading
    rows, vocab = 20, 9000
    c, random = logits_of(30, rows, vocab)
    want = check(c, random, top_p=0.8)
    dev, u = c.cuda(), random.cuda()
    got = [torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(4)]
    wrong = []
    torch.cuda.synchronize()

    def work(i):
        stream = torch.cuda.Stream()
        try:
            for _ in range(20):
                ov.op_sample(dev, u, got[i], top_p=0.8, stream=stream)
                if i % 2:  # refused calls of one thread leave the others' alone
                    with pytest.raises(ov.GeneratorError, match="top_p"):
                        ov.op_sample(dev, u, got[i], top_p=float("nan"), stream=stream)
            stream.synchronize()
        except BaseException as e:
            wrong.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
    for g in got:
        np.testing.assert_array_equal(g.cpu(), want)
