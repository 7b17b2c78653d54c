"""The cache's and the log probabilities' entry points refuse what their
kernels do not cover before any GPU is touched: the messages, on the CPU."""
import ctypes

import pytest

import omnivoice_amd as ov

HERE = 0x10000  # an aligned address that a refused call never reads


def cache(**over):
    f = dict(data=HERE, scales=HERE, blocks=8, block_tokens=32, kv_heads=8, head_dim=128)
    f.update(over)
    return ov._KvCache(**f)


def sequences(**over):
    f = dict(tables=HERE, lengths=HERE, begins=HERE, count=2, table_width=4, rows=10)
    f.update(over)
    return ov._KvSequences(**f)


def refused(fn, *args):
    err = ctypes.create_string_buffer(256)
    status = getattr(ov.lib(), fn)(*args, err, len(err))
    assert status == ov.OVG_ERROR
    return err.value.decode()


BAD_POOLS = [
    (dict(data=None), "null pool"), (dict(scales=None), "null pool"),
    (dict(data=HERE + 8), "16-byte aligned"), (dict(block_tokens=48), "block_tokens"),
    (dict(block_tokens=8), "block_tokens"), (dict(head_dim=96), "head_dim"),
    (dict(kv_heads=0), "kv_heads"), (dict(blocks=0), "blocks"), (dict(blocks=2 ** 31), "blocks")]
BAD_SEQUENCES = [
    (dict(tables=None), "null"), (dict(lengths=None), "null"), (dict(begins=None), "null"),
    (dict(count=-1), "count"), (dict(count=2 ** 21), "count"), (dict(table_width=0), "table_width"),
    (dict(table_width=2 ** 28), "table_width"), (dict(rows=-1), "rows"),
    (dict(rows=2 ** 25), "rows")]


@pytest.mark.parametrize("fn,prefix", [("ovg_op_cache_write", "cache write: "),
                                       ("ovg_op_cache_read", "cache read: ")])
def test_write_and_read_refuse(fn, prefix):
    def call(c, s, k=HERE, v=HERE, ks=1024, vs=1024, kind=0):
        return refused(fn, c, s, k, v, ks, vs, kind, None)
    for over, word in BAD_POOLS:
        message = call(cache(**over), sequences())
        assert message.startswith(prefix) and word in message, message
    for over, word in BAD_SEQUENCES:
        assert word in call(cache(), sequences(**over))
    assert "null" in call(cache(), sequences(), k=None)
    assert "null" in call(cache(), sequences(), v=None)
    assert "stride" in call(cache(), sequences(), ks=1023)
    assert "stride" in call(cache(), sequences(), vs=0)
    assert "type" in call(cache(), sequences(), kind=3)
    assert "type" in call(cache(), sequences(), kind=-1)
    assert "null" in call(None, sequences())
    assert "null" in call(cache(), None)


def test_attention_refuses():
    def call(c, s, q=HERE, o=HERE, qs=2048, os=2048, heads=16, scale=0.1, kind=0, space=None,
             size=0):
        return refused("ovg_op_cache_attention", c, s, q, o, qs, os, heads, scale, 1, kind,
                       space, size, None)
    for over, word in BAD_POOLS:
        message = call(cache(**over), sequences())
        assert message.startswith("cache attention: ") and word in message, message
    for over, word in BAD_SEQUENCES:
        assert word in call(cache(), sequences(**over))
    assert "null" in call(cache(), sequences(), q=None)
    assert "null" in call(cache(), sequences(), o=None)
    assert "heads" in call(cache(), sequences(), heads=12, qs=4096, os=4096)
    assert "heads" in call(cache(), sequences(), heads=4)
    assert "heads" in call(cache(), sequences(), heads=8 * 65, qs=2 ** 20, os=2 ** 20)
    assert "stride" in call(cache(), sequences(), qs=2047)
    assert "stride" in call(cache(), sequences(), os=100)
    assert "scale" in call(cache(), sequences(), scale=float("inf"))
    assert "scale" in call(cache(), sequences(), scale=float("nan"))
    assert "scale" in call(cache(), sequences(), scale=-3e38)  # its log2(e)-fold is not
    assert "type" in call(cache(), sequences(), kind=2)


def test_logprobs_refuse():
    def call(logits=HERE, uncond=None, rows=4, vocab=100, stride=100, u_stride=100, g=0.0,
             mask=-1, tokens=HERE, top=3, logprob=HERE, entropy=HERE, ids=HERE, best=HERE,
             kind=2, space=None, size=0):
        return refused("ovg_op_token_logprobs", logits, uncond, rows, vocab, stride, u_stride, g,
                       mask, tokens, top, logprob, entropy, ids, best, kind, space, size, None)
    assert call(logits=None) == "token logprobs: null pointer"
    assert "rows" in call(rows=-1)
    assert "rows" in call(rows=2 ** 23 + 1)
    assert "vocab" in call(vocab=0)
    assert "vocab" in call(vocab=2 ** 31, stride=2 ** 32)
    assert "stride" in call(stride=99)
    assert "stride" in call(uncond=HERE, u_stride=99)
    assert "top" in call(top=33)
    assert "top" in call(top=-1)
    assert "mask_id" in call(mask=-2)
    assert "mask_id" in call(mask=2 ** 31)
    assert "guidance" in call(g=float("nan"))
    assert "go together" in call(tokens=None)
    assert "go together" in call(logprob=None)
    assert "null" in call(ids=None)
    assert "null" in call(best=None)
    assert "type" in call(kind=7)


def test_nothing_to_do_is_no_error():
    err = ctypes.create_string_buffer(256)
    L = ov.lib()
    assert L.ovg_op_cache_write(cache(), sequences(rows=0), None, None, 1024, 1024, 0, None, err,
                                256) == ov.OVG_OK
    assert L.ovg_op_cache_attention(cache(), sequences(count=0, tables=None, lengths=None,
                                                       begins=None),
                                    None, None, 2048, 2048, 16, 0.1, 0, 0, None, 0, None, err,
                                    256) == ov.OVG_OK
    assert L.ovg_op_token_logprobs(None, None, 0, 10, 10, 10, 0.0, -1, None, 0, None, None, None,
                                   None, 2, None, 0, None, err, 256) == ov.OVG_OK


def test_workspace_queries_refuse_what_their_calls_refuse():
    L = ov.lib()

    def attention(c, s, heads=16):
        return L.ovg_op_cache_attention_workspace(c, s, heads)
    long = sequences(count=1, rows=1, table_width=300)
    assert attention(cache(), long) > 0
    assert attention(cache(), sequences(rows=0)) == 0
    for over, _ in BAD_POOLS:
        assert attention(cache(**over), long) == -1
    for over, _ in BAD_SEQUENCES:
        assert attention(cache(), sequences(**over)) == -1
    assert attention(None, long) == -1
    assert attention(cache(), None) == -1
    for heads in (-16, 0, 4, 12, 8 * 64 + 1, 8 * 65, 2 ** 40):
        assert attention(cache(), long, heads) == -1, heads
    logprobs = L.ovg_op_token_logprobs_workspace
    assert logprobs(1, 151936, 4) > 0
    assert logprobs(0, 151936, 4) == 0
    for args in ((-1, 100, 4), (2 ** 23 + 1, 100, 4), (1, 0, 4), (1, 2 ** 31, 4), (1, 100, -1),
                 (1, 100, 33)):
        assert logprobs(*args) == -1, args


@pytest.mark.parametrize("stream", [None, 0, HERE])
def test_host_tensors_are_refused(stream):
    torch = pytest.importorskip("torch")
    pool = ov.KVCache.empty(4, 1, 128, 32, device="cpu")
    seq = ov.KVSequences(torch.zeros((1, 300), dtype=torch.int32),
                         torch.tensor([9000], dtype=torch.int32),
                         torch.tensor([0, 1], dtype=torch.int32))
    q, k = torch.zeros((1, 2, 128)).half(), torch.zeros((1, 1, 128)).half()
    assert ov.op_cache_attention_workspace(pool, seq, 1, 2) > 0  # the call would take one
    logits, ids = torch.zeros((1, 151936)), torch.zeros((1, 4), dtype=torch.int32)
    for call in (lambda: ov.op_cache_write(pool, seq, k, k, stream=stream),
                 lambda: ov.op_cache_read(pool, seq, k, k, stream=stream),
                 lambda: ov.op_cache_attention(pool, seq, q, q, stream=stream),
                 lambda: ov.op_token_logprobs(logits, None, None, None, ids, torch.zeros((1, 4)),
                                              stream=stream)):
        with pytest.raises(ov.GeneratorError, match="needs tensors of a GPU, got cpu"):
            call()
