"""Argument checks of ikl_sample_tokens, ikl_qk_norm_rope_append_kv and
ikl_copy_blocks: refused before anything is launched, so they run without a
GPU (pointers are addresses that nothing reads)."""

import ctypes

import pytest

from inferkernellab_amd import _lib

P = 1 << 20  # an aligned address


def _sample(**kw):
    a = _lib.SampleArgs()
    a.logits = a.uniform = a.tokens = P
    a.rows, a.vocab, a.logits_stride, a.dtype = 4, 100, 100, _lib.IKL_BF16
    a.temperature = a.top_p = 1.0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(vocab=0), dict(vocab=_lib.SAMPLE_MAX_VOCAB + 1), dict(dtype=3),
                                 dict(dtype=9), dict(logits=0), dict(uniform=0), dict(tokens=0), dict(logits=P + 1),
                                 dict(uniform=P + 2), dict(tokens=P + 4), dict(top_k_rows=P, top_k_type=5),
                                 dict(rows=1 << 31)], ids=str)
def test_sample_refuses(bad):
    lib = _lib.load()
    assert lib.ikl_sample_tokens(ctypes.byref(_sample(**bad)), None) in (_lib.IKL_EINVAL, _lib.IKL_EUNSUPPORTED)
    assert "sample" in _lib.last_error()


def test_sample_of_no_rows_and_workspace_sizes():
    lib = _lib.load()
    assert lib.ikl_sample_tokens(None, None) == _lib.IKL_EINVAL
    assert lib.ikl_sample_tokens(ctypes.byref(_sample(rows=0, logits=0, uniform=0, tokens=0)), None) == _lib.IKL_OK
    assert lib.ikl_sample_workspace_size(ctypes.byref(_sample())) >= 0
    for bad in (dict(rows=-1), dict(vocab=0), dict(vocab=_lib.SAMPLE_MAX_VOCAB + 1)):
        assert lib.ikl_sample_workspace_size(ctypes.byref(_sample(**bad))) < 0


def _norm_rope(weights=None, **kw):
    args = _lib.QKNormRopeArgs()
    a = args.rope
    for name in ("query", "query_out", "key", "value", "cos", "sin", "slots", "k_cache", "v_cache"):
        setattr(a, name, P)
    a.num_tokens, a.num_blocks, a.block_size, a.num_heads, a.num_kv_heads, a.head_dim = 3, 4, 16, 4, 2, 64
    a.dtype = _lib.IKL_BF16
    args.q_weight = args.k_weight = P
    args.eps = 1e-6
    for k, v in (weights or {}).items():
        setattr(args, k, v)
    for k, v in kw.items():
        setattr(a, k, v)
    return args


@pytest.mark.parametrize("bad", [dict(num_tokens=-1), dict(num_tokens=1 << 31), dict(head_dim=0), dict(block_size=0),
                                 dict(key=0), dict(cos=0), dict(slots=0), dict(query=0), dict(query_out=0),
                                 dict(slot_type=4), dict(dtype=3), dict(head_dim=72 + 4), dict(head_dim=2048),
                                 dict(key=P + 8), dict(q_stride_h=3), dict(cache_dtype=_lib.IKL_FP8_E4M3),
                                 dict(weights=dict(q_weight=0)), dict(weights=dict(k_weight=0)),
                                 dict(weights=dict(eps=-1.0)), dict(weights=dict(eps=float("nan"))),
                                 dict(weights=dict(q_weight=P + 2)), dict(weights=dict(k_weight_stride_h=3))], ids=str)
def test_norm_rope_refuses(bad):
    lib = _lib.load()
    assert lib.ikl_qk_norm_rope_append_kv(ctypes.byref(_norm_rope(**bad)), None) in (_lib.IKL_EINVAL,
                                                                                     _lib.IKL_EUNSUPPORTED)
    assert "norm rope append" in _lib.last_error()


def test_norm_rope_of_no_tokens():
    lib = _lib.load()
    assert lib.ikl_qk_norm_rope_append_kv(None, None) == _lib.IKL_EINVAL
    assert lib.ikl_qk_norm_rope_append_kv(ctypes.byref(_norm_rope(num_tokens=0)), None) == _lib.IKL_OK


def _copy(from_, to, **kw):
    a = _lib.CopyBlocksArgs()
    a.base[0] = a.base[1] = P
    for n in range(2):
        a.page_bytes[n] = a.stride_block[n] = 4096
        a.stride_layer[n] = 4096 * 8
    a.num_tensors, a.num_layers, a.num_blocks = 2, 2, 8
    a.num_pairs, a.pairs_on_host, a.index_type = len(from_), 1, _lib.IKL_I32
    keep = ((ctypes.c_int32 * max(1, len(from_)))(*from_), (ctypes.c_int32 * max(1, len(to)))(*to))
    a.src, a.dst = ctypes.addressof(keep[0]), ctypes.addressof(keep[1])
    for k, v in kw.items():
        setattr(a, k, v)
    return a, keep


@pytest.mark.parametrize("src,dst,message", [([0], [8], "invalid block id"), ([-1], [1], "invalid block id"),
                                             ([0, 1], [5, 5], "written twice"), ([0, 1], [1, 2], "read and written"),
                                             ([3], [3], "read and written"), ([0, 4], [4, 5], "read and written")])
def test_copy_refuses_pairs(src, dst, message):
    a, keep = _copy(src, dst)
    assert _lib.load().ikl_copy_blocks(ctypes.byref(a), None) == _lib.IKL_EINVAL
    assert message in _lib.last_error()


@pytest.mark.parametrize("bad", [dict(num_pairs=-1), dict(num_tensors=0), dict(num_tensors=5), dict(num_layers=0),
                                 dict(num_blocks=0), dict(num_blocks=1 << 31), dict(index_type=2), dict(src=0),
                                 dict(dst=0)], ids=str)
def test_copy_refuses_arguments(bad):
    a, keep = _copy([0], [1], **bad)
    assert _lib.load().ikl_copy_blocks(ctypes.byref(a), None) == _lib.IKL_EINVAL
    assert "copy blocks" in _lib.last_error()


@pytest.mark.parametrize("pairs,layers", [(1 << 31, 1), (1 << 34, 1 << 30), ((1 << 63) - 1, 2)])
def test_copy_refuses_more_pages_than_a_launch_holds(pairs, layers):
    """Also where their number wraps round 64 bits (16 Gi pairs of 2^30 layers: to 0)."""
    a, keep = _copy([0], [1], num_pairs=pairs, num_layers=layers, pairs_on_host=0)
    assert _lib.load().ikl_copy_blocks(ctypes.byref(a), None) == _lib.IKL_EINVAL
    assert "too many pages" in _lib.last_error()


def test_copy_of_nothing():
    lib = _lib.load()
    assert lib.ikl_copy_blocks(None, None) == _lib.IKL_EINVAL
    a, keep = _copy([], [])
    assert lib.ikl_copy_blocks(ctypes.byref(a), None) == _lib.IKL_OK
    a, keep = _copy([0], [1])
    a.base[1] = 0
    assert lib.ikl_copy_blocks(ctypes.byref(a), None) == _lib.IKL_EINVAL
    a, keep = _copy([0], [1])
    a.page_bytes[0] = 0
    assert lib.ikl_copy_blocks(ctypes.byref(a), None) == _lib.IKL_EINVAL


def test_struct_layouts_match_the_header():
    import re
    from pathlib import Path

    text = (Path(__file__).resolve().parents[1] / "include" / "ikl_paged.h").read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, cls in (("ikl_qk_norm_rope_args", _lib.QKNormRopeArgs), ("ikl_copy_blocks_args", _lib.CopyBlocksArgs),
                      ("ikl_sample_args", _lib.SampleArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, flags=re.S).group(1)
        fields = []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            names = decl.split(None, 2)[2] if decl.startswith("const") else decl.split(None, 1)[1]
            fields += [re.sub(r"[\s*]|\[\w+\]", "", n) for n in names.split(",")]
        assert fields == [f[0] for f in cls._fields_], name
