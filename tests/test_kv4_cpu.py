"""4-bit KV cache operators: argument checks, which need no GPU (every refusal
comes before the first CUDA call)."""
import ctypes

import pytest

BASE = 1 << 20  # never dereferenced: the calls below are refused on the host


def _cache(**kw):
    import qwen3_b200 as q
    f = dict(k_w=BASE, k_s=2 * BASE, k_b=3 * BASE, v_w=4 * BASE, v_s=5 * BASE, v_b=6 * BASE, batch=2, kv_heads=2,
             max_pos=64, head_dim=128)
    f.update(kw)
    return q.Kv4(*f.values())


def _refused(call, kind=None, text=""):
    import qwen3_b200 as q
    with pytest.raises(kind or q.Error) as e:
        call()
    assert e.value.code in (q.QW_ERR_INVALID_ARG, q.QW_ERR_UNSUPPORTED)
    assert text in e.value.message


@pytest.mark.parametrize("bad,text", [(dict(k_w=0), "16-byte"), (dict(v_b=6 * BASE + 8), "16-byte"),
                                      (dict(head_dim=96), "head_dim"), (dict(head_dim=256), "head_dim"),
                                      (dict(max_pos=0), "max_pos"), (dict(max_pos=40), "max_pos"),
                                      (dict(max_pos=-16), "max_pos"), (dict(batch=0), "batch"),
                                      (dict(kv_heads=0), "kv_heads")])
def test_bad_caches_are_refused_by_every_operator(bad, text):
    import qwen3_b200 as q
    c, ok = _cache(**bad), _cache()
    far = _cache(**{k: 100 * BASE * (i + 1) for i, k in enumerate(("k_w", "k_s", "k_b", "v_w", "v_s", "v_b"))})
    _refused(lambda: q.kv4_append(c, BASE, BASE, 1, BASE), text=text)
    _refused(lambda: q.kv4_read(c, BASE, BASE, 1), text=text)
    _refused(lambda: q.kv4_attention_scratch_bytes(c, 1, 4), text=text)
    _refused(lambda: q.kv4_attention(c, BASE, BASE, 1, 4, 1.0, BASE, BASE, 1 << 30), text=text)
    _refused(lambda: q.kv4_evict_scratch_bytes(c, 8), text=text)
    _refused(lambda: q.kv4_evict(c, far, BASE, BASE, BASE, BASE, 8, 0, BASE, 1 << 30), text=text)
    _refused(lambda: q.kv4_evict(ok, c, BASE, BASE, BASE, BASE, 8, 0, BASE, 1 << 30), text=text)


def test_append_and_read_refusals():
    import qwen3_b200 as q
    c = _cache()
    _refused(lambda: q.kv4_append(c, None, BASE, 1, BASE))
    _refused(lambda: q.kv4_append(c, BASE, None, 1, BASE))
    _refused(lambda: q.kv4_append(c, BASE, BASE, 1, None), text="seq_len")
    _refused(lambda: q.kv4_append(c, BASE + 1, BASE, 1, BASE), text="aligned")
    for S in (0, -1, (1 << 24) + 1):
        _refused(lambda: q.kv4_append(c, BASE, BASE, S, BASE), text="S must")
        _refused(lambda: q.kv4_read(c, BASE, BASE, S), text="S must")
    _refused(lambda: q.kv4_read(c, 0, 0, 1))
    _refused(lambda: q.kv4_read(c, BASE + 8, BASE, 1), text="16-byte")
    assert q.lib().qw_kv4_append(None, BASE, None, BASE, None, 1, BASE, None, None, None) == q.QW_ERR_INVALID_ARG


def test_attention_refusals():
    import qwen3_b200 as q
    c = _cache()

    def call(q_ptr=BASE, out=BASE, S=1, heads=4, scale=1.0, seq=BASE, scratch=BASE, **kw):
        return lambda: q.kv4_attention(c, q_ptr, out, S, heads, scale, seq, scratch, 1 << 30, **kw)

    _refused(call(q_ptr=None))
    _refused(call(out=None))
    _refused(call(seq=None))
    _refused(call(scratch=None))
    _refused(call(heads=3), text="heads")
    _refused(call(heads=0), text="heads")
    _refused(call(S=0), text="S must")
    _refused(call(scale=float("nan")), text="scale")
    _refused(call(scale=float("inf")), text="scale")
    _refused(call(q_ptr=BASE + 2), text="16-byte")
    _refused(call(scratch=BASE + 4), text="16-byte")
    _refused(call(mass_ptr=BASE), text="out may be q only")
    _refused(call(S=2, q_strides=(1024, 512, 128), out_strides=(2048, 1024, 128)), text="out may be q only")
    _refused(call(S=1 << 24, heads=128), text="2^30")
    _refused(call(q_strides=(512, 513, 128)), text="strides")
    _refused(call(out_strides=(512, 512, 4)), text="strides")
    _refused(call(out_strides=(0, 512, 128)), text="zero stride")
    _refused(call(out_strides=(512, 512, 0)), text="zero stride")
    _refused(lambda: q.kv4_attention_scratch_bytes(c, 1, 5), text="heads")
    assert q.lib().qw_kv4_attention_scratch(ctypes.byref(c), 1, 4, None) == q.QW_ERR_INVALID_ARG


def test_evict_refusals():
    import qwen3_b200 as q
    src = _cache()
    dst = _cache(**{k: 100 * BASE * (i + 1) for i, k in enumerate(("k_w", "k_s", "k_b", "v_w", "v_s", "v_b"))})
    m0, m1 = 50 * BASE, 60 * BASE

    def call(s=src, d=dst, ms=m0, md=m1, seq=BASE, new=BASE, keep=8, recent=2, scratch=BASE, nbytes=1 << 30):
        return lambda: q.kv4_evict(s, d, ms, md, seq, new, keep, recent, scratch, nbytes)

    _refused(call(ms=None))
    _refused(call(md=None))
    _refused(call(seq=None))
    _refused(call(new=None))
    _refused(call(scratch=None))
    _refused(call(keep=0), text="keep")
    _refused(call(keep=65), text="keep")
    _refused(call(recent=-1), text="recent")
    _refused(call(recent=9), text="recent")
    _refused(call(nbytes=16), text="scratch")
    other = dict(zip(("k_w", "k_s", "k_b", "v_w", "v_s", "v_b"), (100 * BASE * (i + 1) for i in range(6))))
    _refused(call(d=_cache(**other, batch=1)), text="differ")
    _refused(call(d=_cache(**other, kv_heads=1)), text="differ")
    _refused(call(d=_cache(**other, head_dim=64)), text="differ")
    # the destination shares some arrays with the source, or lies across one
    _refused(call(d=src), text="overlap")             # in place, but the weights go elsewhere
    _refused(call(md=m0), text="overlap")             # elsewhere, but the weights in place
    _refused(call(d=_cache(k_w=BASE + 16)), text="overlap")
    _refused(call(d=_cache(max_pos=32), md=m0), text="overlap")  # the same arrays under another layout
    _refused(lambda: q.kv4_evict_scratch_bytes(src, 0))


@pytest.mark.parametrize("max_pos", [(1 << 30) + 16, (1 << 31) - 32, (1 << 31) - 16])
def test_caches_whose_positions_do_not_fit_tile_counts_are_refused(max_pos):
    """The tile behind the last position would be counted past 2^31 - 1, and read past the arrays."""
    import qwen3_b200 as q
    c, ok = _cache(batch=1, kv_heads=1, head_dim=64, max_pos=max_pos), _cache(batch=1, kv_heads=1, head_dim=64)
    _refused(lambda: q.kv4_append(c, BASE, BASE, 1, BASE), text="2^30")
    _refused(lambda: q.kv4_read(c, BASE, BASE, 1), text="2^30")
    _refused(lambda: q.kv4_attention_scratch_bytes(c, 1, 4), text="2^30")
    _refused(lambda: q.kv4_attention(c, BASE, BASE, 1, 4, 1.0, BASE, BASE, 1 << 30), text="2^30")
    _refused(lambda: q.kv4_evict_scratch_bytes(c, 8), text="2^30")
    _refused(lambda: q.kv4_evict(c, ok, BASE, BASE, BASE, BASE, 8, 0, BASE, 1 << 30), text="2^30")
    _refused(lambda: q.kv4_evict(ok, c, BASE, BASE, BASE, BASE, 8, 0, BASE, 1 << 30), text="2^30")
