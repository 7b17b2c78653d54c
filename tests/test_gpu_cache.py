"""The 8-bit key/value cache against a plain restatement in 64 bits: codes and
scales bit for bit, what is read back bit for bit, and the attention within
the roundings it makes."""
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
# Half a step of each type, relative to the value.
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def _e4m3():
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    x = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    x = np.where((c & 127) == 127, np.nan, x)
    return np.where(c >= 128, -x, x)


E4M3 = _e4m3()


def round_e4m3(x):
    """|x| <= 448 to the nearest e4m3 value, ties to even, exactly."""
    x = np.asarray(x, dtype=np.float64)
    _, e = np.frexp(x)
    step = np.ldexp(1.0, np.maximum(e - 4, -9))
    return np.rint(x / step) * step


def scale_for(amax):
    """The smallest power of two, 2^-100 or more, with amax <= 448 scale."""
    m, e = np.frexp(amax)
    return np.ldexp(1.0, np.where(m > 0, np.maximum(e - 9 + (m > 0.875), -100), -100))


def code_index(block, dim):
    """Index in a block's codes of (token, dim): of keys, of values."""
    t, d = np.arange(block)[:, None], np.arange(dim)
    g, t = t // 16 * 16 * dim, t % 16
    return (g + d // 16 * 256 + t * 16 + d % 16,
            g + d // 64 * 1024 + t // 4 * 256 + d % 16 * 16 + d // 16 % 4 * 4 + t % 4)


class Plain:
    """The pool in 64 bits: codes' values [blocks][heads][2][token][dim] and
    scales [blocks][heads][2]."""

    def __init__(self, cache):
        data = cache.data.cpu().numpy()
        index = code_index(cache.block_tokens, cache.head_dim)
        self.block = cache.block_tokens
        self.codes = np.stack([E4M3[data[:, :, h]][:, :, index[h]] for h in (0, 1)], 2)
        self.scales = cache.scales.cpu().numpy().astype(np.float64)

    def write(self, table, length, k, v):
        """k, v [n][heads][dim], the last tokens of a sequence of `length`."""
        n, B = len(k), self.block
        start = length - n
        for b in range(max(start, 0) // B, -(-length // B)):
            if b >= len(table) or not 0 <= table[b] < len(self.codes):
                continue
            page, lo, hi = table[b], max(start, b * B, 0), min(length, (b + 1) * B)
            if lo >= hi:
                continue
            for half, x in ((0, k), (1, v)):
                x = x[lo - start:hi - start].transpose(1, 0, 2).astype(np.float64)
                for h in range(x.shape[0]):
                    held = self.codes[page, h, half]
                    kept = lo > b * B
                    old = self.scales[page, h, half] if kept else 0.0
                    if not np.isfinite(x[h]).all() or np.isnan(old):
                        self.scales[page, h, half] = np.nan
                        held[lo - b * B:] = 0.0
                        continue
                    s = max(scale_for(np.abs(x[h]).max()), old)
                    if kept:
                        held[:lo - b * B] = round_e4m3(held[:lo - b * B] * (old / s))
                    held[lo - b * B:hi - b * B] = round_e4m3(x[h] / s)
                    held[hi - b * B:] = 0.0
                    self.scales[page, h, half] = s

    def read(self, table, first, last):
        """Keys and values [token][head][dim] at positions first .. last - 1."""
        out = []
        for half in (0, 1):
            rows = []
            for p in range(first, last):
                b = p // self.block
                if p < 0 or b >= len(table) or not 0 <= table[b] < len(self.codes):
                    rows.append(np.zeros(self.codes.shape[1:2] + self.codes.shape[4:]))
                else:
                    rows.append(self.codes[table[b], :, half, p % self.block] *
                                self.scales[table[b], :, half][:, None])
            out.append(np.stack(rows) if rows else
                       np.zeros((0,) + self.codes.shape[1:2] + self.codes.shape[4:]))
        return out

    def there(self, table, length):
        b = np.arange(length) // self.block
        pages = np.array([table[i] if i < len(table) else -1 for i in b], dtype=np.int64)
        return (pages >= 0) & (pages < len(self.codes))


def same(cache, plain):
    got = Plain(cache)
    np.testing.assert_array_equal(got.scales, plain.scales)
    np.testing.assert_array_equal(got.codes, plain.codes)


def sequences(tables, lengths, begins):
    def i32(x):
        return torch.tensor(np.asarray(x, dtype=np.int32)).cuda()
    return ov.KVSequences(i32(tables), i32(lengths), i32(begins))


def tables_of(rng, lengths, block, spare=2, width=None):
    """Shuffled blocks for every sequence, -1 behind them; and the pool's size."""
    need = [-(-max(n, 1) // block) for n in lengths]
    ids = rng.permutation(sum(need) + spare)
    out = np.full((len(lengths), width or max(need)), -1, dtype=np.int32)
    for i, n in enumerate(need):
        out[i, :n] = ids[sum(need[:i]):sum(need[:i]) + n]
    return out, sum(need) + spare


def filled(rng, blocks, heads, dim, block, loud=1.0):
    """A pool with random codes (no NaN) and scales."""
    cache = ov.KVCache.empty(blocks, heads, dim, block)
    data = rng.integers(0, 256, cache.data.shape, dtype=np.uint8)
    data[(data & 127) == 127] = 0
    scales = np.ldexp(1.0, rng.integers(-10, -5, cache.scales.shape)) * loud
    cache.data.copy_(torch.from_numpy(data))
    cache.scales.copy_(torch.from_numpy(scales.astype(np.float32)))
    return cache


def tensor(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(TYPES[dtype]).cuda()


def np64(t):
    return t.detach().double().cpu().numpy()


# ------------------------------------------------------------------ write and read

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_write_then_read_matches_plain(dim, block, dtype):
    """Ragged prompts, appended tokens of several loudnesses over block edges, a
    sequence without new tokens and one written again from the middle."""
    rng = np.random.default_rng(dim + block)
    heads = 3
    lengths = np.array([1, block, block + 1, 3 * block - 1, 5, 2 * block + 7])
    table, blocks = tables_of(rng, lengths + 80, block)
    cache = ov.KVCache.empty(blocks, heads, dim, block)
    plain = Plain(cache)

    def step(new, total, loud):
        begins = np.concatenate([[0], np.cumsum(new)])
        shape = (begins[-1], heads, dim)
        k, v = (tensor(rng.standard_normal(shape) * loud, dtype) for _ in range(2))
        seq = sequences(table, total, begins)
        ov.op_cache_write(cache, seq, k, v)
        for i in range(len(new)):
            rows = slice(begins[i], begins[i + 1])
            plain.write(table[i], total[i], np64(k)[rows], np64(v)[rows])
        same(cache, plain)
        back = [torch.full(shape, 9.0, dtype=TYPES[dtype], device="cuda") for _ in range(2)]
        ov.op_cache_read(cache, seq, *back)
        want = [np.concatenate([plain.read(table[i], total[i] - new[i], total[i])[half]
                                for i in range(len(new))]) for half in (0, 1)]
        for b, w in zip(back, want):
            assert torch.equal(b.cpu(), torch.from_numpy(w).to(TYPES[dtype]))

    step(lengths, lengths, 1.0)
    step(np.array([1, 1, 0, 1, 2, 40]), lengths + [1, 1, 0, 1, 2, 40], 30.0)  # louder
    total = lengths + [1, 1, 0, 1, 2, 40]
    step(np.array([1] * 6), total + 1, 0.01)  # quieter: the scales stay
    step(np.array([1, 9, 2, 17, 4, 39]), total + 1, 3.0)  # written again


def test_every_rounding_and_the_scales_borders():
    """Every fp16 magnitude as a key, in blocks whose scale is one (their loudest
    token is 448); and loudest values on both sides of 448 times a power of two."""
    dim, block = 128, 32
    x = np.arange(0, 0x7C00, dtype=np.uint16).view(np.float16).astype(np.float32)
    x = np.concatenate([x[x <= 448], -x[x <= 448]])
    n = -(-len(x) // ((block - 1) * dim))
    body = np.zeros(n * (block - 1) * dim, np.float32)
    body[:len(x)] = x
    k = np.full((n, block, 1, dim), 448, np.float32)
    k[:, 1:, 0] = body.reshape(n, block - 1, dim)
    k = k.reshape(n * block, 1, dim)
    v = k[:, :, ::-1].copy()
    cache = ov.KVCache.empty(n, 1, dim, block)
    plain = Plain(cache)
    table = np.arange(n, dtype=np.int32)[None]
    ov.op_cache_write(cache, sequences(table, [n * block], [0, n * block]), tensor(k, "f16"),
                      tensor(v, "f16"))
    plain.write(table[0], n * block, k, v)
    assert (plain.scales == 1).all()
    same(cache, plain)
    edges = [448, 448.25, 447.75, 449, 500, 896, 897, 1e-30, 0.0, 2.0 ** -133, 3e38, 1e-20,
             448 * 2.0 ** -100, 449 * 2.0 ** -100]
    cache = ov.KVCache.empty(len(edges), 1, dim, 16)
    plain = Plain(cache)
    k = np.linspace(-1, 1, len(edges) * 16 * dim).astype(np.float32).reshape(-1, 16, 1, dim)
    k = (k * np.array(edges, np.float32)[:, None, None, None]).reshape(-1, 1, dim)
    k[::16, 0, 5] = edges
    table = np.arange(len(edges), dtype=np.int32)[None]
    t = torch.from_numpy(k).cuda()
    ov.op_cache_write(cache, sequences(table, [len(k)], [0, len(k)]), t, t)
    plain.write(table[0], len(k), k, k)
    same(cache, plain)


def test_write_without_blocks_rows_or_tokens():
    """Bad table entries, positions past the table, more rows than tokens, rows
    before the first and behind the last sequence, empty sequences: what has no
    place is dropped or zero, everything else is as it was."""
    rng = np.random.default_rng(5)
    dim, block, heads = 64, 16, 2
    table = np.array([[3, -1, 2], [99, 4, 2 ** 31 - 1], [5, 6, 7], [8, 0, 0], [1, -5, 9]])
    lengths = np.array([40, 30, 70, 3, 0])
    begins = np.array([4, 24, 44, 74, 80, 85])  # the fourth has 6 rows and 3 tokens
    rows = 90
    cache = filled(rng, 10, heads, dim, block)
    plain = Plain(cache)
    k, v = (tensor(rng.standard_normal((rows, heads, dim)), "f16") for _ in range(2))
    seq = sequences(table, lengths, begins)
    ov.op_cache_write(cache, seq, k, v)
    for i in range(5):
        sl = slice(begins[i], begins[i + 1])
        plain.write(table[i], lengths[i], np64(k)[sl], np64(v)[sl])
    same(cache, plain)
    back = [torch.full((rows, heads, dim), 9.0, dtype=torch.float32, device="cuda")
            for _ in range(2)]
    ov.op_cache_read(cache, seq, *back)
    for half in (0, 1):
        want = np.full((rows, heads, dim), 9.0)
        for i in range(5):
            n = begins[i + 1] - begins[i]
            want[begins[i]:begins[i + 1]] = plain.read(table[i], lengths[i] - n,
                                                       lengths[i])[half]
        np.testing.assert_array_equal(np64(back[half]), want)


def test_begins_past_the_rows_are_clamped():
    rng = np.random.default_rng(6)
    dim, block = 64, 16
    cache = filled(rng, 8, 1, dim, block)
    before = cache.data.clone()
    x = tensor(rng.standard_normal((10, 1, dim)), "f16")
    seq = sequences([[0, 1], [2, 3], [4, 5]], [20, 20, 20], [-7, 8, 500, 2 ** 31 - 1])
    ov.op_cache_write(cache, seq, x, x)
    changed = (cache.data != before).flatten(1).any(1).cpu().numpy()
    assert not changed[[4, 5, 6, 7]].any() and changed[[0, 1, 2, 3]].any()
    ov.op_cache_read(cache, seq, x, x)
    out = torch.full((10, 2, dim), 9.0, dtype=torch.float16, device="cuda")
    ov.op_cache_attention(cache, seq, tensor(rng.standard_normal((10, 2, dim)), "f16"), out)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all() and (out != 9).any(-1).all()


@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_block_with_no_number_is_nan(where, bad):
    """One infinity or NaN: its head's block of that half is NaN until it is
    written from its first token again, nothing else is touched."""
    rng = np.random.default_rng(8)
    dim, block, heads, n = 64, 16, 3, 60
    table, blocks = tables_of(rng, [n], block)
    cache = ov.KVCache.empty(blocks, heads, dim, block)
    plain = Plain(cache)
    x = {h: rng.standard_normal((n, heads, dim)).astype(np.float32) for h in "kv"}
    x[where][21, 1, 7] = bad
    k, v = tensor(x["k"], "f16"), tensor(x["v"], "f16")
    ov.op_cache_write(cache, sequences(table, [n], [0, n]), k, v)
    plain.write(table[0], n, np64(k), np64(v))
    same(cache, plain)
    assert np.isnan(plain.scales).sum() == 1
    # Tokens 30 .. 59 again: token 21's block keeps tokens and stays NaN.
    ov.op_cache_write(cache, sequences(table, [n], [0, n - 30]), k[30:], v[30:])
    plain.write(table[0], n, np64(k)[30:], np64(v)[30:])
    same(cache, plain)
    assert np.isnan(plain.scales).sum() == 1
    k = torch.nan_to_num(k, 0.0, 0.0, 0.0)
    v = torch.nan_to_num(v, 0.0, 0.0, 0.0)
    ov.op_cache_write(cache, sequences(table, [n], [0, n - 16]), k[16:], v[16:])
    plain.write(table[0], n, np64(k)[16:], np64(v)[16:])
    same(cache, plain)
    assert np.isfinite(plain.scales).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("offset", [0, 1, 3, 8])
def test_fused_rows_at_any_alignment(dtype, offset):
    """k and v as views into fused q|k|v rows of an odd stride, from a base that
    is aligned to one element only."""
    rng = np.random.default_rng(offset)
    dim, block, heads, n = 128, 32, 2, 45
    width = 6 * dim + offset
    flat = tensor(rng.standard_normal(n * width + 16), dtype)
    fused = flat[offset:offset + n * width].view(n, width)
    k = fused[:, 2 * dim:4 * dim].view(n, heads, dim)
    v = fused[:, 4 * dim:6 * dim].view(n, heads, dim)
    table, blocks = tables_of(rng, [n], block)
    cache = ov.KVCache.empty(blocks, heads, dim, block)
    plain = Plain(cache)
    seq = sequences(table, [n], [0, n])
    ov.op_cache_write(cache, seq, k, v)
    plain.write(table[0], n, np64(k), np64(v))
    same(cache, plain)
    before = flat.clone()
    ov.op_cache_read(cache, seq, k, v)
    want = before.clone()
    wv = want[offset:offset + n * width].view(n, width)
    for half, a in ((0, 2 * dim), (1, 4 * dim)):
        wv[:, a:a + 2 * dim] = torch.from_numpy(
            plain.read(table[0], 0, n)[half].reshape(n, -1)).to(TYPES[dtype]).cuda()
    assert torch.equal(flat, want)


# ------------------------------------------------------------------ attention

def attend64(plain, table, length, q, group, scale, causal):
    """o, and the sum of |weight * value| that bounds its roundings, in 64 bits;
    and the largest score magnitude that a query's products sum to."""
    n = len(q)
    k, v = plain.read(table, 0, length)
    there = plain.there(table, length)
    o = np.zeros(q.shape)
    mass = np.zeros(q.shape)
    sums = np.zeros(q.shape[:2])
    for h in range(q.shape[1]):
        kk, vv = k[:, h // group], v[:, h // group]
        s = q[:, h] @ kk.T * scale
        seen = np.broadcast_to(there, (n, length)).copy()
        if causal:
            seen &= np.arange(length)[None] <= (length - n + np.arange(n))[:, None]
        s = np.where(seen, s, -np.inf)
        top = s.max(1, keepdims=True, initial=-np.inf)
        w = np.exp(s - np.where(np.isfinite(top), top, 0))
        total = w.sum(1, keepdims=True)
        w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
        o[:, h] = w @ vv
        mass[:, h] = w @ np.abs(vv)
        if length:
            sums[:, h] = (np.abs(q[:, h]) @ np.abs(kk).T * abs(scale) * seen).max(1)
    return o, mass, sums


def check_attention(cache, seq_np, q, out, group, dtype, scale, causal, touched=None):
    """Every row within the roundings: scores in float32 (dim + 8 of them), the
    probabilities and the output to the type, sums in float32. The output's own
    last step: half one; twice the probabilities', whose sum is rounded too."""
    tables, lengths, begins = seq_np
    plain = Plain(cache)
    got, q64 = np64(out), np64(q)
    half = HALF_STEP[dtype]
    capacity = tables.shape[1] * cache.block_tokens
    for i, length in enumerate(lengths):
        rows = slice(begins[i], begins[i + 1])
        n = begins[i + 1] - begins[i]
        if n == 0:
            continue
        # Rows before position 0 of a causal call see nothing.
        o, mass, sums = attend64(plain, tables[i], length, q64[rows], group, scale, causal)
        value = np.abs(plain.read(tables[i], 0, min(length, capacity))[1]).max(initial=0.0)
        score = (cache.head_dim + 8) * 2.0 ** -24 * sums[..., None]
        # Weights that are subnormal in fp16 are off by up to 2^-25 each.
        tiny = length * 2.0 ** -25 * value if dtype == "f16" else 0.0
        tol = (2 * half + 2 * score + 2.0 ** -18) * mass + half * np.abs(o) + tiny + 2.0 ** -25
        err = np.abs(got[rows] - o)
        assert np.isfinite(got[rows]).all()
        assert (err <= tol).all(), (i, n, length, float((err / tol).max()))


def attention_case(seed, new, lengths, heads, group, dim, block, dtype, causal, width=None,
                   loud=1.0, scale=None):
    rng = np.random.default_rng(seed)
    new, lengths = np.array(new), np.array(lengths)
    table, blocks = tables_of(rng, lengths, block, width=width)
    cache = filled(rng, blocks, heads, dim, block, loud)
    begins = np.concatenate([[0], np.cumsum(new)])
    q = tensor(rng.standard_normal((begins[-1], heads * group, dim)), dtype)
    out = torch.full_like(q, 9.0)
    scale = dim ** -0.5 if scale is None else scale
    ov.op_cache_attention(cache, sequences(table, lengths, begins), q, out, scale=scale,
                          causal=causal)
    check_attention(cache, (table, lengths, begins), q, out, group, dtype, scale, causal)
    return cache, (table, lengths, begins), q, out


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_of_single_tokens(dtype, dim, block, causal):
    attention_case(1, [1] * 9, [1, 2, 15, 16, 17, 33, 250, 511, 1027], 2, 2, dim, block, dtype,
                   causal)


@pytest.mark.parametrize("new,lengths,heads,group,dim,block,dtype,causal", [
    ([5, 1, 0, 7], [5, 600, 40, 300], 4, 1, 128, 32, "f16", True),
    ([8, 8, 3], [900, 30, 64], 2, 8, 64, 16, "bf16", True),
    ([60, 17, 33], [400, 17, 700], 2, 2, 128, 32, "f16", False),
    ([100, 1, 257], [100, 1, 900], 1, 4, 128, 64, "bf16", True),
    ([300, 130], [300, 1100], 2, 2, 128, 16, "f16", True),
    ([129, 64, 65], [129, 640, 65], 1, 3, 64, 32, "bf16", False),
    ([40], [45], 1, 64, 64, 16, "f16", True),
    ([513], [2000], 1, 2, 64, 64, "f16", False),
    ([1], [9000], 1, 1, 128, 16, "f16", True),
    ([2, 4], [20011, 5000], 1, 2, 128, 64, "bf16", True),
    ([700], [700], 2, 5, 128, 32, "f16", True),
])
def test_attention_matches_plain(new, lengths, heads, group, dim, block, dtype, causal):
    attention_case(2, new, lengths, heads, group, dim, block, dtype, causal)


@pytest.mark.parametrize("new,lengths", [([3] * 30, [40] * 30), ([1] * 200, [70] * 200),
                                         ([150] * 6, [333] * 6)])
def test_attention_of_many_sequences(new, lengths):
    attention_case(3, new, lengths, 2, 2, 64, 16, "f16", True)


@pytest.mark.parametrize("new,lengths,heads,group,dim,block,dtype,causal", [
    ([250, 1, 0, 131, 64], [400, 300, 9, 131, 70], 16, 9, 128, 32, "f16", True),
    ([250, 33, 131], [300, 1000, 131], 16, 12, 128, 16, "bf16", False),
    ([300, 2, 130], [310, 40, 200], 32, 10, 64, 64, "bf16", True),
    ([300, 2, 130], [310, 40, 200], 32, 10, 64, 16, "f16", False),
    ([520, 40], [1700, 1100], 16, 15, 128, 64, "f16", True),
])
def test_attention_of_rows_that_fill_the_device(new, lengths, heads, group, dim, block, dtype,
                                                causal):
    """A tile to a wave: tiles that end inside a work-group, sequences without rows.
    Two kv heads are compared."""
    rng = np.random.default_rng(25)
    table, blocks = tables_of(rng, lengths, block)
    cache = filled(rng, blocks, heads, dim, block)
    begins = np.concatenate([[0], np.cumsum(new)])
    q = tensor(rng.standard_normal((begins[-1], heads * group, dim)), dtype)
    out = torch.full_like(q, 9.0)
    ov.op_cache_attention(cache, sequences(table, lengths, begins), q, out, causal=causal)
    assert torch.isfinite(out).all() and (out != 9).any(-1).all()
    for head in (1, heads - 1):
        one = ov.KVCache(cache.data[:, head:head + 1].contiguous(),
                         cache.scales[:, head:head + 1].contiguous(), block, dim)
        rows = slice(head * group, (head + 1) * group)
        check_attention(one, (table, np.array(lengths), begins), q[:, rows], out[:, rows], group,
                        dtype, dim ** -0.5, causal)


def test_more_sequences_than_a_launch_holds():
    """70000 sequences of one token each over eight shared blocks, and some of
    none: against the same rows in calls of their own."""
    rng = np.random.default_rng(20)
    count, dim, block, heads = 70000, 64, 16, 1
    table = rng.integers(0, 8, (count, 1))
    lengths = rng.integers(1, 17, count)
    new = np.where(rng.random(count) < 0.01, 0, 1)
    begins = np.concatenate([[0], np.cumsum(new)])
    cache = filled(rng, 8, heads, dim, block)
    q = tensor(rng.standard_normal((begins[-1], 1, dim)), "f16")
    out = torch.full_like(q, 9.0)
    ov.op_cache_attention(cache, sequences(table, lengths, begins), q, out, causal=True)
    again = torch.full_like(q, 9.0)
    for a in range(0, count, 25000):
        rows = slice(begins[a], begins[min(a + 25000, count)])
        ov.op_cache_attention(
            cache, sequences(table[a:a + 25000], lengths[a:a + 25000],
                             begins[a:a + 25001] - begins[a]), q[rows], again[rows], causal=True)
    assert torch.equal(out, again) and (out != 9).any(-1).all()
    pick = rng.permutation(np.flatnonzero(new))[:300]
    check_attention(cache, (table[pick], lengths[pick], np.arange(301)), q[begins[pick]],
                    out[begins[pick]], 1, "f16", dim ** -0.5, True)
    k = tensor(rng.standard_normal((begins[-1], 1, dim)), "f16")
    v = torch.empty_like(k)
    ov.op_cache_read(cache, sequences(table, lengths, begins), k, v)
    plain = Plain(cache)
    at = np.stack([plain.read(table[i], lengths[i] - 1, lengths[i])[1][0] for i in pick])
    np.testing.assert_array_equal(np64(v[begins[pick]]), at)


def test_long_tables_of_small_blocks():
    """20000 tokens in blocks of 16: each wave goes through several windows of the
    table, some of whose blocks are missing or NaN behind the rows' sight."""
    rng = np.random.default_rng(21)
    for new, dtype in ((1, "f16"), (30, "bf16")):
        table, blocks = tables_of(rng, [20000], 16)
        table[0, rng.permutation(1250)[:200]] = -1
        cache = filled(rng, blocks, 1, 64, 16)
        cache.scales[:, :, 1] *= torch.from_numpy(
            np.ldexp(1.0, rng.integers(0, 8, (blocks, 1))).astype(np.float32)).cuda()
        q = tensor(rng.standard_normal((new, 2, 64)), dtype)
        out = torch.empty_like(q)
        seq_np = (table, np.array([20000]), np.array([0, new]))
        ov.op_cache_attention(cache, sequences(*seq_np), q, out, causal=True)
        check_attention(cache, seq_np, q, out, 2, dtype, 0.125, True)


@pytest.mark.parametrize("new", [2, 60, 200])
def test_attention_rows_that_see_nothing(new):
    """More rows than tokens (causal: the first ones come before position 0),
    sequences of no tokens, tables without a block: zero. Rows of no sequence:
    as they were."""
    rng = np.random.default_rng(9)
    dim, block, heads, group = 64, 16, 2, 2
    table = np.array([[0, 1, 2, 3], [-1, -1, 99, -1], [4, -1, 5, 6], [7, 8, -3, 9]])
    lengths = np.array([new - 1, 50, 60, 0])
    begins = 3 + np.arange(5) * new
    rows = begins[-1] + 5
    cache = filled(rng, 10, heads, dim, block)
    q = tensor(rng.standard_normal((rows, heads * group, dim)), "f16")
    for causal in (False, True):
        out = torch.full_like(q, 9.0)
        ov.op_cache_attention(cache, sequences(table, lengths, begins), q, out, causal=causal)
        got = np64(out)
        assert (got[:3] == 9).all() and (got[begins[-1]:] == 9).all()
        assert (got[begins[1]:begins[2]] == 0).all()  # no blocks
        assert (got[begins[3]:begins[4]] == 0).all()  # no tokens
        if causal:
            assert (got[begins[0]] == 0).all()        # before position 0
        at = np.minimum(lengths, table.shape[1] * block)
        if new - 1 <= 4 * block:
            check_attention(cache, (table[[0, 2]], at[[0, 2]],
                                    np.array([0, new, 2 * new])),
                            torch.cat([q[begins[0]:begins[1]], q[begins[2]:begins[3]]]),
                            torch.cat([out[begins[0]:begins[1]], out[begins[2]:begins[3]]]),
                            group, "f16", dim ** -0.5, causal)


@pytest.mark.parametrize("new", [1, 6, 40, 200])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_nan_stays_where_it_is_seen(new, dtype):
    """A NaN block of keys or of values makes NaN the rows that see a token of
    it, in its heads, and no other: not rows before it, not the other heads;
    a NaN behind the end of the sequence, none."""
    rng = np.random.default_rng(10)
    dim, block, heads, group = 64, 16, 4, 2
    total = 400
    table, blocks = tables_of(rng, [total], block)
    cache = filled(rng, blocks, heads, dim, block)
    start = total - new
    bad = start + new // 2  # a position among the new tokens
    cache.scales[table[0, bad // block], 1, 0] = float("nan")
    cache.scales[table[0, bad // block], 2, 1] = float("nan")
    q = tensor(rng.standard_normal((new, heads * group, dim)), dtype)
    out = torch.full_like(q, 9.0)
    seq = sequences(table, [total], [0, new])
    ov.op_cache_attention(cache, seq, q, out, causal=True)
    nan = torch.isnan(out).cpu().numpy()
    # The first row that sees a token of the block: the one at its first token.
    first = max(bad // block * block - start, 0)
    want = np.zeros(nan.shape, dtype=bool)
    want[first:, 2:6] = True
    np.testing.assert_array_equal(nan, want)
    clean = filled(rng, blocks, heads, dim, block)
    clean.data.copy_(cache.data)
    clean.scales.copy_(torch.nan_to_num(cache.scales, 1.0))
    other = torch.full_like(q, 9.0)
    ov.op_cache_attention(clean, seq, q, other, causal=True)
    keep = torch.from_numpy(~want).cuda()
    assert torch.equal(out[keep], other[keep])
    # The sequence cut before the block: nothing of it is left.
    cut = bad // block * block
    n = min(new, cut)
    ov.op_cache_attention(cache, sequences(table, [cut], [0, n]), q[:n], out[:n])
    assert torch.isfinite(out[:n]).all()


@pytest.mark.parametrize("new", [1, 40, 200])
def test_attention_infinite_queries_stay_in_their_rows(new):
    rng = np.random.default_rng(11)
    table, blocks = tables_of(rng, [300], 32)
    cache = filled(rng, blocks, 2, 128, 32)
    q = tensor(rng.standard_normal((new, 4, 128)), "f16")
    seq = sequences(table, [300], [0, new])
    clean = torch.empty_like(q)
    ov.op_cache_attention(cache, seq, q, clean, causal=True)
    at = new // 2
    bad = q.clone()
    bad[at, 1, 5] = float("inf")
    bad[at, 2, 6] = float("nan")
    out = torch.empty_like(q)
    ov.op_cache_attention(cache, seq, bad, out, causal=True)
    nan = torch.isnan(out).cpu()
    want = torch.zeros_like(nan)
    want[at, 1:3] = True
    assert torch.equal(nan, want)
    assert torch.equal(out[~want.cuda()], clean[~want.cuda()])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 3, 200])
def test_attention_of_loud_and_quiet_blocks(dtype, new):
    """Values whose loudness changes by 2^30 (bf16; 2^12 in fp16) from block to
    block, up to fp16's largest, and keys of one loud block that takes it all."""
    rng = np.random.default_rng(12)
    dim, block, heads, total = 64, 16, 2, 320
    table, blocks = tables_of(rng, [total], block)
    cache = filled(rng, blocks, heads, dim, block)
    span = 30 if dtype == "bf16" else 12
    cache.scales[:, :, 1] = torch.from_numpy(
        np.ldexp(1.0, rng.integers(-span, 1, (blocks, heads))).astype(np.float32)).cuda() * 64
    cache.scales[table[0, 3], 0, 0] = 1.0
    q = tensor(rng.standard_normal((new, heads * 2, dim)), dtype)
    out = torch.empty_like(q)
    seq_np = (table, np.array([total]), np.array([0, new]))
    ov.op_cache_attention(cache, sequences(*seq_np), q, out, causal=True)
    check_attention(cache, seq_np, q, out, 2, dtype, dim ** -0.5, True)


@pytest.mark.parametrize("new", [1, 9, 150])
def test_attention_growing_scores(new):
    """Scores that rise along the keys, so that every step finds a new maximum,
    and scores that fall, so that none after the first does; a scale of zero."""
    rng = np.random.default_rng(13)
    dim, block, total = 64, 16, 800
    table, blocks = tables_of(rng, [total], block)
    for order in (1, -1):
        cache = ov.KVCache.empty(blocks, 1, dim, block)
        k = np.zeros((total, 1, dim), np.float32)
        k[:, 0, 0] = np.arange(total)[::order] * 0.5
        v = rng.standard_normal((total, 1, dim)).astype(np.float32)
        ov.op_cache_write(cache, sequences(table, [total], [0, total]), tensor(k, "f16"),
                          tensor(v, "f16"))
        q = torch.zeros((new, 2, dim), dtype=torch.float16, device="cuda")
        q[:, 0, 0] = 1.0
        q[:, 1, 0] = 30.0
        seq_np = (table, np.array([total]), np.array([0, new]))
        for scale in (0.125, 0.0, -0.125):
            out = torch.empty_like(q)
            ov.op_cache_attention(cache, sequences(*seq_np), q, out, scale=scale)
            check_attention(cache, seq_np, q, out, 2, "f16", scale, False)


def test_attention_strided_queries_and_output():
    rng = np.random.default_rng(14)
    dim, block, heads, group, n, total = 128, 32, 2, 2, 70, 300
    table, blocks = tables_of(rng, [total], block)
    cache = filled(rng, blocks, heads, dim, block)
    for offset in (0, 1, 5):
        width = (heads * group + 4) * dim + offset
        flat = tensor(rng.standard_normal(n * width + 8), "bf16")
        fused = flat[offset:offset + n * width].view(n, width)
        q = fused[:, :heads * group * dim].view(n, heads * group, dim)
        store = torch.full((n * (width + 3) + 8,), 9.0, dtype=torch.bfloat16, device="cuda")
        rows = store[offset:offset + n * (width + 3)].view(n, width + 3)
        out = rows[:, :heads * group * dim].view(n, heads * group, dim)
        for m in (1, 4, n):
            seq_np = (table, np.array([total]), np.array([0, m]))
            out.fill_(9.0)
            ov.op_cache_attention(cache, sequences(*seq_np), q, out)
            check_attention(cache, seq_np, q, out, group, "bf16", dim ** -0.5, False)
            left = store.clone()
            left[offset:offset + n * (width + 3)].view(n, width + 3)[:m, :heads * group * dim] = 9
            assert (left == 9).all()


@pytest.mark.parametrize("new,lengths", [([1, 1, 1], [70, 900, 33]), ([1], [9000]),
                                         ([40, 3, 129], [100, 3, 640]), ([200], [6000])])
def test_attention_in_place(new, lengths):
    """Into the queries' own rows: whole, and in splits that are joined."""
    rng = np.random.default_rng(24)
    dim, block, heads, group = 128, 32, 2, 3
    table, blocks = tables_of(rng, lengths, block)
    cache = filled(rng, blocks, heads, dim, block)
    seq = sequences(table, lengths, np.concatenate([[0], np.cumsum(new)]))
    q = tensor(rng.standard_normal((sum(new), heads * group, dim)), "f16")
    out = torch.empty_like(q)
    ov.op_cache_attention(cache, seq, q, out, causal=True)
    ov.op_cache_attention(cache, seq, q, q, causal=True)
    assert torch.equal(out, q)


def test_attention_single_tokens_do_not_depend_on_their_batch():
    """A sequence's rows are the same bits alone and among others."""
    rng = np.random.default_rng(15)
    lengths = [37, 5000, 700, 16]
    cache, (table, lengths, begins), q, out = attention_case(
        15, [1, 2, 2, 1], lengths, 2, 2, 128, 32, "f16", True)
    for i in range(4):
        rows = slice(begins[i], begins[i + 1])
        alone = torch.empty_like(q[rows])
        ov.op_cache_attention(cache, sequences(table[i:i + 1], lengths[i:i + 1],
                                               [0, begins[i + 1] - begins[i]]),
                              q[rows].contiguous(), alone, causal=True)
        err = (alone.double() - out[rows].double()).abs().max().item()
        # Another split of the keys may round otherwise; nothing more.
        assert err <= 4 * HALF_STEP["f16"] * out[rows].abs().max().item()


def test_same_bits_every_time():
    cache, seq_np, q, out = attention_case(16, [1, 5, 90], [3000, 900, 1500], 2, 2, 128, 32,
                                           "f16", True)
    for _ in range(3):
        again = torch.empty_like(out)
        ov.op_cache_attention(cache, sequences(*seq_np), q, again, causal=True)
        assert torch.equal(again, out)


# ------------------------------------------------------------------ streams, graphs, workspaces

def test_serving_steps_in_a_graph():
    """Write, attend, project and rate in one captured step, replayed while the
    lengths grow on the device: every step equals the eager calls'."""
    rng = np.random.default_rng(17)
    dim, block, heads, group, count, vocab = 128, 16, 2, 2, 3, 200
    start = np.array([30, 1, 500], np.int32)
    table, blocks = tables_of(rng, start + 40, block)
    pools = [ov.KVCache.empty(blocks, heads, dim, block) for _ in range(2)]
    begins = np.concatenate([[0], np.cumsum(start)])
    k, v = (tensor(rng.standard_normal((begins[-1], heads, dim)), "f16") for _ in range(2))
    for pool in pools:
        ov.op_cache_write(pool, sequences(table, start, begins), k, v)
    head = tensor(rng.standard_normal((vocab, heads * group * dim)) * 0.05, "f16")
    warm = torch.empty((count, vocab), dtype=torch.float32, device="cuda")
    ov.op_linear_noalloc(torch.zeros((count, heads * group * dim), dtype=torch.float16,
                                     device="cuda"), head, warm)

    def buffers():
        return dict(q=torch.zeros((count, heads * group, dim), dtype=torch.float16, device="cuda"),
                    k=torch.zeros((count, heads, dim), dtype=torch.float16, device="cuda"),
                    v=torch.zeros((count, heads, dim), dtype=torch.float16, device="cuda"),
                    out=torch.zeros((count, heads * group, dim), dtype=torch.float16,
                                    device="cuda"),
                    logits=torch.zeros((count, vocab), device="cuda"),
                    tokens=torch.tensor([3, 0, 150], dtype=torch.int32, device="cuda"),
                    logprob=torch.zeros(count, device="cuda"),
                    entropy=torch.zeros(count, device="cuda"),
                    ids=torch.zeros((count, 4), dtype=torch.int32, device="cuda"),
                    best=torch.zeros((count, 4), device="cuda"),
                    seq=sequences(table, start, np.arange(count + 1)))

    def step(pool, b, **spaces):
        b["seq"].lengths.add_(1)
        ov.op_cache_write(pool, b["seq"], b["k"], b["v"])
        ov.op_cache_attention(pool, b["seq"], b["q"], b["out"], causal=True,
                              workspace=spaces.get("attention"))
        ov.op_linear_noalloc(b["out"].view(count, -1), head, b["logits"])
        ov.op_token_logprobs(b["logits"], b["tokens"], b["logprob"], b["entropy"], b["ids"],
                             b["best"], workspace=spaces.get("logprobs"))

    eager, caught = buffers(), buffers()
    spaces = dict(
        attention=torch.empty(max(16, ov.op_cache_attention_workspace(
            pools[1], caught["seq"], count, heads * group)), dtype=torch.uint8, device="cuda"),
        logprobs=torch.empty(1 << 16, dtype=torch.uint8, device="cuda"))
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step(pools[1], caught, **spaces)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(20):
        for name in ("q", "k", "v"):
            x = torch.randn(eager[name].shape, device="cuda").half()
            eager[name].copy_(x)
            caught[name].copy_(x)
        step(pools[0], eager)
        graph.replay()
        torch.cuda.synchronize()
        for name in ("out", "logits", "logprob", "entropy", "ids", "best"):
            assert torch.equal(eager[name], caught[name]), name
        assert torch.equal(pools[0].data, pools[1].data)
        assert torch.equal(pools[0].scales, pools[1].scales)
        assert torch.equal(eager["seq"].lengths, caught["seq"].lengths)


def test_calls_on_a_stream_of_their_own():
    """On a side stream behind slow work, without any wait by the caller, and
    with a workspace that the call takes for itself."""
    rng = np.random.default_rng(18)
    dim, block, n = 128, 32, 3000
    table, blocks = tables_of(rng, [n], block)
    cache = ov.KVCache.empty(blocks, 2, dim, block)
    k, v = (tensor(rng.standard_normal((n, 2, dim)), "f16") for _ in range(2))
    q = tensor(rng.standard_normal((1, 4, dim)), "f16")
    out = torch.empty_like(q)
    seq_np = (table, np.array([n]), np.array([0, 1]))
    whole, one = sequences(table, [n], [0, n]), sequences(*seq_np)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    big = torch.zeros(1 << 26, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(10):
            big.add_(1.0)
    ov.op_cache_write(cache, whole, k, v, stream=side)
    ov.op_cache_attention(cache, one, q, out, stream=side.cuda_stream)
    junk = torch.full((1 << 22,), 255, dtype=torch.uint8, device="cuda")  # may reuse its memory
    side.synchronize()
    del junk
    plain = Plain(cache)
    assert (plain.scales > 0)[table[0]].all()
    check_attention(cache, seq_np, q, out, 2, "f16", dim ** -0.5, False)


def test_a_new_workspace_is_its_streams_own():
    """Memory that the current stream still uses must not serve another one."""
    side = torch.cuda.Stream()
    device = torch.device("cuda", torch.cuda.current_device())
    for stream, handle in ((side, side.cuda_stream), (side.cuda_stream, side.cuda_stream),
                           (None, 0)):
        at, size, keep = ov._workspace(None, 5 << 20, device, stream)
        assert size == 5 << 20
        owner = [s["stream"] for s in torch.cuda.memory_snapshot()
                 if s["address"] <= at < s["address"] + s["total_size"]]
        assert owner == [handle]


def test_a_workspace_of_the_callers():
    cache, seq_np, q, out = attention_case(19, [1, 1], [6000, 9000], 1, 2, 128, 32, "f16", True)
    seq = sequences(*seq_np)
    size = ov.op_cache_attention_workspace(cache, seq, 2, 2)
    space = torch.full((size + 64,), 255, dtype=torch.uint8, device="cuda")
    again = torch.empty_like(out)
    ov.op_cache_attention(cache, seq, q, again, causal=True, workspace=space[:size + 16])
    assert torch.equal(out, again)
    assert (space[size:] == 255).all()
    if size:
        with pytest.raises(ov.GeneratorError, match="^cache attention: workspace"):
            ov.op_cache_attention(cache, seq, q, again, workspace=space[:size - 1])


def test_tensors_are_checked():
    cache = ov.KVCache.empty(4, 2, 64, 16)
    seq = sequences([[0, 1]], [5], [0, 5])
    x = torch.zeros((5, 2, 64), dtype=torch.float16, device="cuda")
    for bad in (x[:, :1], x.transpose(1, 2), x.double(), x[:, :, ::2], x.cpu(), x[:4],
                x.float(), x[:1].expand(5, 2, 64)):
        with pytest.raises(ov.GeneratorError):
            ov.op_cache_write(cache, seq, x, bad)
    q = torch.zeros((5, 4, 64), dtype=torch.float16, device="cuda")
    for a, b in ((q.float(), q.float()), (q, q[:4]), (q, q.bfloat16()), (q[:, :3], q[:, :3]),
                 (q[0], q[0]), (q.cpu(), q.cpu())):
        with pytest.raises(ov.GeneratorError):
            ov.op_cache_attention(cache, seq, a, b)
    with pytest.raises(ov.GeneratorError):
        ov.op_cache_attention(cache, seq, q, q, scale=float("nan"))
    with pytest.raises(ov.GeneratorError):
        ov.KVCache(cache.data.cpu(), cache.scales, 16, 64)
    with pytest.raises(ov.GeneratorError):
        ov.KVSequences(seq.tables.long(), seq.lengths, seq.begins)
    # No rows, no sequences: nothing to do.
    ov.op_cache_write(cache, seq, x[:0], x[:0])
    ov.op_cache_attention(cache, seq, q[:0], q[:0])
    none = sequences(np.zeros((0, 1)), [], [0])
    ov.op_cache_read(cache, none, x, x)
    torch.cuda.synchronize()


# ------------------------------------------------------------------ blocks that are not there

def gaps_of(table, lengths, block, blocks):
    """The same sequences over a pool whose first block is nobody's, with a part of
    each one's blocks missing (names outside the pool); and the blocks left unnamed."""
    table = np.where(table >= 0, table + 1, table)
    for i, length in enumerate(lengths):
        n = -(-length // block)
        table[i, n // 6:n // 2] = no_names(n // 2 - n // 6)
    return table, np.setdiff1d(np.arange(blocks + 1), table)


def no_names(n):
    return np.resize(np.array([-1, 2 ** 31 - 1, -2 ** 31], dtype=np.int64), n).astype(np.int32)


def spoil(cache, blocks):
    """What memory that nobody wrote may hold: codes and scales that are no numbers."""
    at = torch.from_numpy(np.asarray(blocks)).cuda()
    cache.data[at] = 255
    cache.scales[at] = float("nan")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("new,lengths", [
    ([1, 1, 1, 1], [1, 17, 45, 200]),    # tiles of 16 rows
    ([1], [9001]),                       # split, some splits without any block
    ([2, 1, 2, 1], [2000, 90, 1500, 16]),
    ([40, 1, 33], [40, 17, 300]),        # tiles of 32 rows
    ([60], [5001]),                      # and split
])
def test_attention_beside_blocks_without_contents(dtype, dim, block, new, lengths):
    """Blocks that no sequence names hold codes and scales that are no numbers, the
    pool's first among them, and some of each sequence's blocks are missing: nothing
    of either reaches a row."""
    rng = np.random.default_rng(block + dim)
    table, blocks = tables_of(rng, lengths, block)
    table, rest = gaps_of(table, lengths, block, blocks)
    cache = filled(rng, blocks + 1, 2, dim, block)
    spoil(cache, rest)
    begins = np.concatenate([[0], np.cumsum(new)])
    q = tensor(rng.standard_normal((begins[-1], 4, dim)), dtype)
    for causal in (False, True):
        out = torch.full_like(q, 9.0)
        ov.op_cache_attention(cache, sequences(table, lengths, begins), q, out, causal=causal)
        check_attention(cache, (table, np.array(lengths), begins), q, out, 2, dtype, dim ** -0.5,
                        causal)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("block", [16, 32, 64])
def test_attention_of_many_rows_beside_blocks_without_contents(dtype, block):
    """The same where a wave takes a tile with all its keys: rows that fill the
    device (at least 2048 tiles of 128 dims over the kv heads, 1024 positions at
    most). Two kv heads are compared."""
    rng = np.random.default_rng(block)
    new, lengths, heads, group, dim = [250, 1, 131, 3], [300, 17, 131, 20], 16, 12, 128
    table, blocks = tables_of(rng, lengths, block)
    table, rest = gaps_of(table, lengths, block, blocks)
    cache = filled(rng, blocks + 1, heads, dim, block)
    spoil(cache, rest)
    begins = np.concatenate([[0], np.cumsum(new)])
    q = tensor(rng.standard_normal((begins[-1], heads * group, dim)), dtype)
    out = torch.full_like(q, 9.0)
    ov.op_cache_attention(cache, sequences(table, lengths, begins), q, out, causal=True)
    assert torch.isfinite(out).all() and (out != 9).any(-1).all()
    for head in (0, heads - 1):
        one = ov.KVCache(cache.data[:, head:head + 1].contiguous(),
                         cache.scales[:, head:head + 1].contiguous(), block, dim)
        rows = slice(head * group, (head + 1) * group)
        check_attention(one, (table, np.array(lengths), begins), q[:, rows], out[:, rows], group,
                        dtype, dim ** -0.5, True)


@pytest.mark.parametrize("block", [16, 32, 64])
def test_a_pool_without_initial_contents(block):
    """Written, attended and read back in a pool of which every byte was 255."""
    rng = np.random.default_rng(31)
    lengths = np.array([1, 16, 17, 33, 64, 65, 130])
    table, blocks = tables_of(rng, lengths, block)
    table = np.where(table >= 0, table + 1, table)
    cache = ov.KVCache.empty(blocks + 1, 2, 64, block)
    spoil(cache, np.arange(blocks + 1))
    begins = np.concatenate([[0], np.cumsum(lengths)])
    k, v = (tensor(rng.standard_normal((begins[-1], 2, 64)), "f16") for _ in range(2))
    q = tensor(rng.standard_normal((begins[-1], 4, 64)), "f16")
    seq = sequences(table, lengths, begins)
    ov.op_cache_write(cache, seq, k, v)
    out, one = torch.full_like(q, 9.0), torch.full_like(q[:len(lengths)], 9.0)
    ov.op_cache_attention(cache, seq, q, out, causal=True)
    check_attention(cache, (table, lengths, begins), q, out, 2, "f16", 0.125, True)
    last = np.arange(len(lengths) + 1)
    ov.op_cache_attention(cache, sequences(table, lengths, last), q[begins[1:] - 1], one)
    check_attention(cache, (table, lengths, last), q[begins[1:] - 1], one, 2, "f16", 0.125, False)
    back = [torch.empty_like(k) for _ in range(2)]
    ov.op_cache_read(cache, seq, *back)
    assert torch.isfinite(back[0]).all() and torch.isfinite(back[1]).all()


# ------------------------------------------------------------------ borders outside the rows

@pytest.mark.parametrize("begins,lengths,rows", [
    ([0, 12], [20], 10), ([0, 30], [40], 17), ([2, 30, 41], [50, 60], 35),
    ([-5, 9, 30], [40, 21], 20), ([-9, 40], [45], 20), ([0, 25], [20], 12),
    ([0, 3, 2 ** 31 - 1], [30, 2 ** 31 - 1], 9), ([0, 2 ** 31 - 1], [40], 9)])
@pytest.mark.parametrize("block", [16, 32])
def test_rows_keep_their_places_where_begins_names_more(begins, lengths, rows, block):
    """Row r of a sequence whose rows end at `end` is its token length - (end - r),
    whichever of its rows there are: written there, read from there, and seeing as
    far. Tokens whose rows are not there are not written."""
    rng = np.random.default_rng(rows)
    heads, dim = 2, 64
    table, blocks = tables_of(rng, [64] * len(lengths), block)
    cache = filled(rng, blocks, heads, dim, block)
    plain = Plain(cache)
    k, v = (tensor(rng.standard_normal((rows, heads, dim)), "f16") for _ in range(2))
    q = tensor(rng.standard_normal((rows, 2 * heads, dim)), "f16")
    seq = sequences(table, lengths, begins)
    ov.op_cache_write(cache, seq, k, v)
    spans = []  # rows, and the place behind the last one's
    for i, length in enumerate(lengths):
        first, last = max(begins[i], 0), min(begins[i + 1], rows)
        spans.append((slice(first, max(first, last)), length - begins[i + 1] + last))
        sl, end = spans[-1]
        if sl.stop > sl.start and end > 0:
            plain.write(table[i], end, np64(k)[sl][-end:], np64(v)[sl][-end:])
    same(cache, plain)
    back = [torch.full((rows, heads, dim), 9.0, dtype=torch.float32, device="cuda")
            for _ in range(2)]
    ov.op_cache_read(cache, seq, *back)
    for half in (0, 1):
        want = np.full((rows, heads, dim), 9.0)
        for i, (sl, end) in enumerate(spans):
            want[sl] = plain.read(table[i], end - (sl.stop - sl.start), end)[half]
        np.testing.assert_array_equal(np64(back[half]), want)
    for causal in (False, True):
        out = torch.full_like(q, 9.0)
        ov.op_cache_attention(cache, seq, q, out, causal=causal)
        got = np64(out)
        for i, (sl, end) in enumerate(spans):
            n = sl.stop - sl.start
            if n == 0:
                continue
            # A causal call's rows see as far as those of a sequence that ends there.
            sees = min(end if causal else lengths[i], 64)
            if sees <= 0:
                assert (got[sl] == 0).all()
                continue
            check_attention(cache, (table[i:i + 1], np.array([sees]), np.array([0, n])), q[sl],
                            out[sl], 2, "f16", dim ** -0.5, causal)


# ------------------------------------------------------------------ the type's largest values

@pytest.mark.parametrize("new,total,heads,group", [
    (1, 900, 1, 2),     # one work-group a head
    (1, 2000, 2, 2),    # few splits, joined by groups of lanes
    (1, 9000, 1, 2),    # many
    (50, 700, 1, 2), (60, 5000, 1, 2), (260, 300, 16, 16)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_attention_of_values_near_the_types_largest(new, total, heads, group, sign):
    """Averages of many values of bfloat16's upper end are finite, though their sums
    are not: 1e38 to 3e38, equal scores and random ones."""
    rng = np.random.default_rng(total)
    dim, block = 128, 32
    table, blocks = tables_of(rng, [total], block)
    cache = ov.KVCache.empty(blocks, heads, dim, block)
    k = rng.standard_normal((total, heads, dim)) * (np.arange(heads)[:, None] > 0)
    v = sign * rng.uniform(1e38, 3e38, (total, heads, dim))
    ov.op_cache_write(cache, sequences(table, [total], [0, total]), tensor(k, "bf16"),
                      tensor(v, "bf16"))
    q = tensor(rng.standard_normal((new, heads * group, dim)), "bf16")
    out = torch.empty_like(q)
    seq_np = (table, np.array([total]), np.array([0, new]))
    ov.op_cache_attention(cache, sequences(*seq_np), q, out, causal=True)
    assert torch.isfinite(out).all()
    for head in sorted({0, heads - 1}):
        one = ov.KVCache(cache.data[:, head:head + 1].contiguous(),
                         cache.scales[:, head:head + 1].contiguous(), block, dim)
        rows = slice(head * group, (head + 1) * group)
        check_attention(one, seq_np, q[:, rows], out[:, rows], group, "bf16", dim ** -0.5, True)


# ------------------------------------------------------------------ batches and tables

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new,lengths,heads,group", [
    ([1, 2, 2, 1], [37, 5000, 700, 16], 2, 2), ([1] * 40, [100 + 7 * i for i in range(40)], 8, 2),
    ([40, 3, 129, 1], [100, 3, 640, 900], 2, 3), ([250, 131, 1, 3], [300, 131, 90, 64], 16, 12)])
def test_a_sequence_has_the_same_bits_beside_any_others(dtype, new, lengths, heads, group):
    """The others' queries, keys and values changed, infinities among them, and all of
    them in another order: the calls are planned alike, so the bits stay."""
    rng = np.random.default_rng(26)
    dim, block = 128, 32
    table, blocks = tables_of(rng, lengths, block)
    cache = filled(rng, blocks, heads, dim, block)
    begins = np.concatenate([[0], np.cumsum(new)])
    q = tensor(rng.standard_normal((begins[-1], heads * group, dim)), dtype)
    out = torch.full_like(q, 9.0)
    ov.op_cache_attention(cache, sequences(table, lengths, begins), q, out, causal=True)
    order = rng.permutation(len(new))
    moved = np.concatenate([np.arange(begins[i], begins[i + 1]) for i in order])
    again = torch.full_like(q, 9.0)
    ov.op_cache_attention(
        cache, sequences(table[order], np.array(lengths)[order],
                         np.concatenate([[0], np.cumsum(np.array(new)[order])])),
        q[torch.from_numpy(moved).cuda()].contiguous(), again, causal=True)
    assert torch.equal(again, out[torch.from_numpy(moved).cuda()])
    for keep in sorted({0, len(new) // 2, len(new) - 1}):
        other = filled(rng, blocks, heads, dim, block, loud=2.0 ** 20)
        mine = torch.from_numpy(table[keep][table[keep] >= 0].astype(np.int64)).cuda()
        other.data[mine], other.scales[mine] = cache.data[mine], cache.scales[mine]
        rows = slice(begins[keep], begins[keep + 1])
        x = torch.full_like(q, float("inf"))
        x[rows] = q[rows]
        ov.op_cache_attention(other, sequences(table, lengths, begins), x, again, causal=True)
        assert torch.equal(again[rows], out[rows])


@pytest.mark.parametrize("new,dtype", [(1, "f16"), (30, "bf16"), (200, "f16")])
@pytest.mark.parametrize("block", [16, 64])
def test_no_numbers_behind_the_rows_sight(new, dtype, block):
    """A long causal sequence whose table goes on behind it, with blocks whose scales
    and codes are no numbers, others missing: the rows are those without them."""
    rng = np.random.default_rng(27)
    total, dim = 20000, 64
    table, blocks = tables_of(rng, [total + 50 * block], block)
    table[0, rng.permutation(total // block)[:100]] = -1
    cache = filled(rng, blocks, 1, dim, block)
    seen = table[0, :-(-total // block)]
    spoil(cache, np.setdiff1d(np.arange(blocks), seen))
    q = tensor(rng.standard_normal((new, 2, dim)), dtype)
    out = torch.full_like(q, 9.0)
    seq_np = (table, np.array([total]), np.array([0, new]))
    ov.op_cache_attention(cache, sequences(*seq_np), q, out, causal=True)
    check_attention(cache, seq_np, q, out, 2, dtype, dim ** -0.5, True)
    # Inside the sequence, behind all rows but the last ones.
    if new > block:
        last = (total - 1) // block
        kept = torch.from_numpy(np.arange(new) < last * block - (total - new)).cuda()
        cache.scales[int(table[0, last])] = float("nan")
        again = torch.full_like(q, 9.0)
        ov.op_cache_attention(cache, sequences(*seq_np), q, again, causal=True)
        assert torch.equal(again[kept], out[kept]) and torch.isnan(again[~kept]).all()


@pytest.mark.parametrize("new,lengths,width,group,dtype", [
    ([1], [430], 4096, 2, "f16"), ([1, 1, 3], [1, 17, 2000], 4096, 2, "bf16"),
    ([40], [100], 2048, 2, "f16"), ([600, 1, 1, 5], [700, 20000, 90, 4000], None, 2, "f16"),
    ([2048, 1], [2048, 9001], None, 1, "bf16")])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_of_wide_tables_and_mixed_calls(new, lengths, width, group, dtype, causal):
    """Tables far wider than their sequences, whose splits are mostly empty, and
    prompts beside single tokens over long sequences."""
    attention_case(28, new, lengths, 1, group, 64, 32, dtype, causal, width=width)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("total", [300, 3000])
def test_attention_of_infinite_scores(new, total):
    """Scores that overflow: -infinity has no weight, a row of nothing else is zero,
    +infinity makes its row NaN."""
    rng = np.random.default_rng(29)
    dim, block = 64, 32
    table, blocks = tables_of(rng, [total], block)
    cache = ov.KVCache.empty(blocks, 1, dim, block)
    k = np.zeros((total, 1, dim), np.float32)
    k[::2, 0, 0] = 100.0   # the first query head's scores there are -infinity
    k[:, 0, 1] = 100.0     # and all of the second's, and the third's +infinity
    v = rng.standard_normal((total, 1, dim))
    ov.op_cache_write(cache, sequences(table, [total], [0, total]), tensor(k, "bf16"),
                      tensor(v, "bf16"))
    q = torch.zeros((new, 4, dim), dtype=torch.bfloat16, device="cuda")
    q[:, 0, 0] = -3e38
    q[:, 1, 1] = -3e38
    q[:, 2, 1] = 3e38
    out = torch.full_like(q, 9.0)
    ov.op_cache_attention(cache, sequences(table, [total], [0, new]), q, out, scale=8.0)
    got = np64(out)
    held = Plain(cache).read(table[0], 0, total)[1][:, 0]
    # Equal weights of one, float32 sums: half a step of the output and 2^-18 of the mass.
    for head, x in ((0, held[1::2]), (3, held)):
        tol = 2.0 ** -8 * np.abs(x.mean(0)) + 2.0 ** -18 * np.abs(x).mean(0)
        assert (np.abs(got[:, head] - x.mean(0)) <= tol).all()
    assert (got[:, 1] == 0).all() and np.isnan(got[:, 2]).all()


@pytest.mark.parametrize("block,dim", [(16, 64), (32, 128)])
def test_offsets_past_32_bits(block, dim):
    """Blocks more than 2^32 bytes into the pool, and rows more than 2^32 elements
    apart: the same as in a small pool and from packed rows."""
    rng = np.random.default_rng(30)
    heads, n = 8, 500
    per = heads * 2 * block * dim
    blocks = (5 << 30) // per
    ids = blocks - 1 - rng.permutation(3000)[:-(-n // block)]
    pool = torch.empty((blocks, heads, 2, block * dim), dtype=torch.uint8, device="cuda")
    big = ov.KVCache(pool, torch.empty((blocks, heads, 2), device="cuda"), block, dim)
    small = ov.KVCache.empty(len(ids), heads, dim, block)
    assert int(ids.min()) * per > 2 ** 32
    k, v = (tensor(rng.standard_normal((n, heads, dim)), "f16") for _ in range(2))
    q = tensor(rng.standard_normal((3, 2 * heads, dim)), "f16")
    flat = torch.empty((2 << 31) + (1 << 20), dtype=torch.float16, device="cuda")
    wide = {h: flat[at:].as_strided((3, h, dim), (1 << 31, dim, 1))
            for at, h in ((0, heads), (1 << 16, 2 * heads))}
    wide[heads].copy_(k[-3:])
    wide[2 * heads].copy_(q)
    got = []
    for cache, table in ((small, np.arange(len(ids))), (big, ids)):
        seq, last = sequences([table], [n], [0, n]), sequences([table], [n], [0, 3])
        ov.op_cache_write(cache, seq, k, v)
        if cache is big:
            ov.op_cache_write(cache, last, wide[heads], v[-3:])
        at = torch.from_numpy(np.asarray(table)).cuda()
        back = [torch.empty_like(k) for _ in range(2)]
        ov.op_cache_read(cache, seq, *back)
        x = q if cache is small else wide[2 * heads]
        out = torch.empty_like(q)
        ov.op_cache_attention(cache, last, x, out, causal=True)
        if cache is big:
            ov.op_cache_read(cache, last, wide[heads], torch.empty_like(k[:3]))
            assert torch.equal(wide[heads], back[0][-3:])
            ov.op_cache_attention(cache, last, x, wide[2 * heads], causal=True)
            assert torch.equal(wide[2 * heads], out)
        got.append([cache.data[at], cache.scales[at], *back, out])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("new,total,heads,group", [
    (1, 300, 1, 2), (1, 9000, 1, 2), (50, 700, 1, 2), (60, 5000, 1, 2), (260, 300, 16, 16)])
@pytest.mark.parametrize("dtype,loud", [("f16", 3e4), ("bf16", 3e4), ("bf16", 1e15)])
@pytest.mark.parametrize("offset", [0.0, 1.0])
def test_attention_of_large_scores(new, total, heads, group, dtype, loud, offset):
    """Finite scores of 1e8 and more, positive or (with an offset) all negative, under
    scales that are no power of two: the keys of the largest share all of the weight,
    the next code's scores being a sixteenth of it away, a thousand and more."""
    rng = np.random.default_rng(33)
    dim, block = 128, 32
    table, blocks = tables_of(rng, [total], block)
    cache = ov.KVCache.empty(blocks, heads, dim, block)
    k = np.zeros((total, heads, dim), np.float32)
    k[..., 0] = loud * (rng.uniform(0.2, 1.0, (total, heads)) - 1.3 * offset)
    v = rng.standard_normal((total, heads, dim))
    ov.op_cache_write(cache, sequences(table, [total], [0, total]), tensor(k, dtype),
                      tensor(v, dtype))
    q = torch.zeros((new, heads * group, dim), dtype=TYPES[dtype], device="cuda")
    q[..., 0] = loud
    q[:, 1::2, 0] *= 0.37
    keys, values = Plain(cache).read(table[0], 0, total)
    for scale in (0.1, 0.113, 0.7):
        out = torch.full_like(q, 9.0)
        ov.op_cache_attention(cache, sequences(table, [total], [0, new]), q, out, scale=scale)
        got = np64(out)
        for head in sorted({0, heads - 1}):
            best = keys[:, head, 0] == keys[:, head, 0].max()
            x = values[best, head]
            # The weights are equal and rounded alike, the sums float32: half a step.
            tol = HALF_STEP[dtype] * np.abs(x.mean(0)) + 2.0 ** -18 * np.abs(x).mean(0) + 2.0 ** -25
            err = np.abs(got[:, head * group:(head + 1) * group] - x.mean(0))
            assert (err <= tol).all(), (scale, head, float(np.nanmax(err / tol)))


@pytest.mark.parametrize("new", [8, 40, 200])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_large_scores_stay_in_their_rows(new, dtype):
    """One row with scores of 1e4 and more, one with scores of infinity: the others'
    bits are those without them."""
    rng = np.random.default_rng(34)
    table, blocks = tables_of(rng, [700], 32)
    cache = filled(rng, blocks, 2, 128, 32)
    q = tensor(rng.standard_normal((new, 4, 128)), dtype)
    seq = sequences(table, [700], [0, new])
    clean, out = torch.empty_like(q), torch.empty_like(q)
    ov.op_cache_attention(cache, seq, q, clean, causal=True)
    bad = q.clone()
    bad[new // 2, 1] *= 1e4
    bad[new // 2, 2, 5] = float("inf")
    ov.op_cache_attention(cache, seq, bad, out, causal=True, scale=128 ** -0.5)
    want = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
    want[new // 2, 1:3] = False
    assert torch.equal(out[want], clean[want])
    assert torch.isfinite(out[new // 2, 1]).all()
