"""What the readings operators refuse, checked on the host (no GPU needed)."""

import ctypes as C

import pytest
import torch

from sheetsage2_refined_b200 import _lib, ops


def sample_args(**kw):
    a = _lib.SampleArgs(logits=16, logits_stride=8, logits_dtype=_lib.S2R_F32, rows=2, vocab=8, uniforms=16,
                        temperature_all=1.0, top_p_all=1.0, tokens=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(logits=None), b"NULL"), (dict(uniforms=None), b"NULL"), (dict(tokens=None), b"NULL"),
    (dict(rows=0), b"rows"), (dict(vocab=0), b"vocab"), (dict(rows=65537), b"65536"), (dict(vocab=524289), b"524288"),
    (dict(logits_dtype=3), b"float32"), (dict(logits_stride=-1), b"stride"), (dict(allowed_stride=-8), b"stride"),
    (dict(temperature_all=-0.5), b"temperature"), (dict(temperature_all=float("nan")), b"temperature"),
    (dict(top_p_all=1.5), b"top_p"), (dict(top_p_all=float("nan")), b"top_p"), (dict(min_p_all=-0.1), b"min_p"),
    (dict(top_k_all=-1), b"top_k"), (dict(logits=18), b"aligned"), (dict(tokens=20), b"aligned"),
    (dict(uniforms=17), b"aligned"), (dict(bias=18), b"aligned"), (dict(top_k=19), b"aligned"),
    (dict(logprobs=22), b"aligned"),
])
def test_sample_entry_point_refuses(change, word):
    lib = _lib.load()
    assert lib.s2r_sample(C.byref(sample_args(**change)), None) == _lib.S2R_EINVAL
    assert word in lib.s2r_last_error()


def test_sample_refuses_null_arguments():
    lib = _lib.load()
    assert lib.s2r_sample(None, None) == _lib.S2R_EINVAL


def test_sample_wrapper_refuses_host_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        ops.sample(torch.zeros(2, 8), torch.zeros(2))


def attention_args(**kw):
    a = _lib.SharedAttentionArgs(
        dtype=_lib.S2R_BF16, rows=2, heads=4, kv_heads=2, head_dim=64, scale=0.125, q=16, q_row_stride=256,
        q_head_stride=64, shared_k=16, shared_v=16, k_token_stride=128, k_head_stride=64, v_token_stride=128,
        v_head_stride=64, shared_tokens=100, out=16, out_row_stride=256, out_head_stride=64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


OWN = dict(own_k=16, own_v=16, own_pages=4, pages_per_row=2, page_table=16, page_table_stride=2, own_len=16)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=_lib.S2R_F32), b"bfloat16"), (dict(rows=0), b"rows"), (dict(rows=65536), b"65535"),
    (dict(heads=5), b"multiple"), (dict(heads=0), b"heads"), (dict(kv_heads=0), b"kv_heads"),
    (dict(heads=8192), b"4096"), (dict(shared_tokens=-1), b"shared_tokens"), (dict(shared_tokens=2**30), b"2^28"),
    (dict(q=None), b"NULL"), (dict(out=None), b"NULL"), (dict(shared_v=None), b"NULL"), (dict(shared_k=24), b"aligned"),
    (dict(k_token_stride=132), b"multiples of 8"), (dict(v_head_stride=65), b"multiples of 8"),
    (dict(k_token_stride=32), b"overlap"), (dict(out_row_stride=32), b"overlap"), (dict(out_head_stride=8), b"overlap"),
    (dict(rows=65535, heads=512), b"2^24"), (dict(v_head_stride=32), b"overlap"), (dict(q_row_stride=-1), b"strides"), (dict(scale=0.0), b"scale"), (dict(scale=float("nan")), b"scale"),
    (dict(scale=float("inf")), b"scale"), (dict(own_k=16), b"go together"), (dict(own_len=16), b"go together"),
    (dict(OWN, own_pages=0), b"own_pages"), (dict(OWN, pages_per_row=0), b"pages_per_row"),
    (dict(OWN, page_table_stride=1), b"page table"), (dict(OWN, own_pages=2**24), b"2^25"), (dict(OWN, own_v=40), b"aligned"),
    (dict(q=17), b"aligned"), (dict(out=33), b"aligned"), (dict(lse=18), b"aligned"), (dict(shared_len=18), b"aligned"),
    (dict(OWN, page_table=18), b"aligned"), (dict(OWN, own_len=18), b"aligned"), (dict(error=18), b"aligned"),
    # rows one head apart, heads one row apart: (0, 1) and (1, 0) of out would be the same place
    (dict(out_row_stride=64, out_head_stride=64), b"overlap"), (dict(out_row_stride=192, out_head_stride=64), b"overlap"),
])
def test_shared_attention_entry_point_refuses(change, word):
    lib = _lib.load()
    assert lib.s2r_shared_attention(C.byref(attention_args(**change)), None) == _lib.S2R_EINVAL
    assert word in lib.s2r_last_error()
    n = C.c_int64(-1)
    assert lib.s2r_shared_attention_workspace(C.byref(attention_args(**change)), C.byref(n)) == _lib.S2R_EINVAL
    assert n.value == -1


def test_shared_attention_refuses_other_head_dims_and_null_arguments():
    lib = _lib.load()
    assert lib.s2r_shared_attention(C.byref(attention_args(head_dim=80)), None) == _lib.S2R_ENOTSUP
    assert lib.s2r_shared_attention(None, None) == _lib.S2R_EINVAL
    assert lib.s2r_shared_attention_workspace(C.byref(attention_args()), None) == _lib.S2R_EINVAL


def test_shared_attention_wrapper_refuses_host_tensors():
    t = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.shared_attention(t, t, t)


def test_sampled_step_and_shared_window_refusals():
    lib = _lib.load()
    assert lib.s2r_step_sampled(None, 1, C.byref(_lib.Sampling()), None) == _lib.S2R_EINVAL
    grammar, weights = _lib.GrammarDesc(kind=1, states=1, table=16), _lib.Weights()
    weights.layers = (_lib.LayerWeights * 1)()
    ctx = C.c_void_p()
    for width, flags, word in ((64, 0, b"width of at least"), (256, 32, b"tensor-core"), (256, 4, b"flag bits")):
        cfg = _lib.Config(vocab_size=512, width=width, layers=1, heads=width // 64, ffn_width=1024, max_tokens=64,
                          batch=1, frames=8, flags=flags)
        rc = lib.s2r_create_shared(C.byref(cfg), C.byref(weights), C.byref(grammar), 0, C.byref(ctx))
        assert rc in (_lib.S2R_ENOTSUP, _lib.S2R_EINVAL) and word in lib.s2r_last_error()


class FakeEngine:
    """Enough of ``BatchDecoder`` for ``decode_readings``: slot s ends after s + 2 polls."""

    def __init__(self, batch, shared=True):
        self.batch, self.shared_window, self.device = batch, shared, "cpu"
        self.loaded, self.left, self.logprob = [False] * batch, [0] * batch, [0.0] * batch
        self.memories, self.polls = [], 0

    def free_slots(self):
        return [s for s in range(self.batch) if not self.loaded[s]]

    def load(self, slot, memory, prefix, stop, frames, logp, target):
        self.memories.append(memory)
        self.loaded[slot], self.left[slot], self.logprob[slot] = True, slot + 2, -float(len(self.memories))

    def run_sampled(self, uniforms, **kw):
        assert uniforms.shape == (4, self.batch) and 0 <= float(uniforms.min()) and float(uniforms.max()) < 1
        self.left = [n - 1 for n in self.left]
        self.polls += 1

    def finished(self):
        return [s for s in range(self.batch) if self.loaded[s] and self.left[s] <= 0]

    def take(self, slot):
        self.loaded[slot] = False
        return [1, 2], "eos"


def test_decode_readings_refills_slots_and_ranks():
    from sheetsage2_refined_b200.shard import Song, decode_readings

    eng = FakeEngine(3)
    got = decode_readings(eng, Song("memory", [1, 3]), 8, poll_every=4)
    assert [r.logprob for r in got] == [-float(i) for i in range(1, 9)]
    assert eng.memories == ["memory"] + [None] * 7  # the window is brought once
    for bad in (dict(readings=0), dict(readings=1, poll_every=0)):
        with pytest.raises(ValueError):
            decode_readings(FakeEngine(2), Song("m"), **bad)
    with pytest.raises(ValueError, match="shared_window"):
        decode_readings(FakeEngine(2, shared=False), Song("m"), 1)
    busy = FakeEngine(2)
    busy.loaded[1] = True
    with pytest.raises(ValueError, match="no slot loaded"):
        decode_readings(busy, Song("m"), 1)
