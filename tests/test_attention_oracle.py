"""CPU checks of the attention operators' plain forms, of the helpers of
consumer_int8.attention and of the C boundary's refusals (no kernel is launched)."""

import ctypes
import re

import numpy as np
import pytest

from oracle import attention as OA
from tests.conftest import HEADER_PATH

ATTENTION_HEADER = HEADER_PATH.parent / "consumer_int8_attention.h"


def test_quantized_values_are_the_nearest():
    """Against a search over all eight magnitudes, with ties to the even code."""
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((64, 128)) * np.exp(rng.standard_normal((64, 1)) * 6)).astype(np.float32)
    x[0, :32] = np.float32([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7] * 4)  # ties at scale 1
    codes, scales = OA.fp4_quantize(x)
    assert scales[0, 0] == 127
    got = OA.fp4_values(codes, scales)
    unit = np.repeat(np.exp2(scales.astype(np.float64) - 127), 32, -1)
    y = np.abs(x.astype(np.float64)) / unit
    distance = np.abs(y[..., None] - OA.E2M1)
    order = np.argsort(distance + np.arange(8) % 2 * 1e-12, -1, kind="stable")[..., 0]
    assert np.array_equal(np.abs(got), OA.E2M1[order] * unit)
    assert np.array_equal(np.signbit(got), np.signbit(x))
    # the scale is the smallest that holds the block, to within what rounds down to 6
    amax = np.abs(x.astype(np.float64)).reshape(64, 4, 32).max(-1)
    assert (amax <= 7 * unit[:, ::32]).all() and (amax > 3.5 * unit[:, ::32]).all()


@pytest.mark.parametrize("value,byte", [(0.0, 2), (2.0**-130, 2), (7 * 2.0**-125, 2),
                                        (7.5 * 2.0**-125, 3), (1.0, 125), (1.75, 125),
                                        (1.7500001, 126), (7.0, 127), (7.0000005, 128),
                                        (2.9e38, 252), (3.0e38, 252), (3.4e38, 252), (np.inf, 255), (np.nan, 255)])
def test_scale_bytes(value, byte):
    assert OA.fp4_scale_bytes(np.float32([value]))[0] == byte


def test_blocks_with_infinities_read_as_nan():
    x = np.ones((1, 64), dtype=np.float32)
    x[0, 40] = -np.inf
    codes, scales = OA.fp4_quantize(x)
    assert list(scales[0]) == [125, 255] and not codes[0, 16:].any()
    values = OA.fp4_values(codes, scales)
    assert (values[0, :32] == 1).all() and np.isnan(values[0, 32:]).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_fp32_form_stays_by_the_formula(interleaved):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((5, 3, 128)).astype(np.float32)
    w = np.exp(rng.standard_normal(128)).astype(np.float32)
    angle = np.arange(50)[:, None] * 0.9 ** np.arange(16)
    table = np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)
    at = np.stack([rng.integers(0, 50, 5) for _ in range(3)])
    axes = rng.integers(0, 3, 16)
    args = (w, 1e-6, table, 32, at, axes, interleaved)
    y, size = OA.norm_rope64(x, *args)
    assert np.all(np.abs(OA.norm_rope32(x, *args) - y) <= size * 18 * 2.0**-24)
    assert np.array_equal(y[..., 32:], OA.norm_rope64(x, w, 1e-6, None, 0, None, None, False)[0][..., 32:])


def test_positions_outside_the_table_are_nan():
    y, _ = OA.norm_rope64(np.ones((3, 1, 64)), None, 0, np.ones((4, 16)), 16, [3, 4, -1], None, False)
    assert np.isfinite(y[0]).all() and np.isnan(y[1:, :, :16]).all() and np.isfinite(y[1:, :, 16:]).all()


def test_attention_of_nothing():
    out, lse, _, _ = OA.attention64(np.ones((2, 4)), np.ones((3, 4)), np.ones((3, 4)), [0, 2], [0, 0], 1.0)
    assert (out[0] == 0).all() and np.isneginf(lse[0])
    assert np.allclose(out[1], 1) and np.isclose(lse[1], 4 + np.log(2))


# ---- the C boundary ---------------------------------------------------------------------


def declared():
    return sorted(set(re.findall(r"^int (ci8_\w+)\(", ATTENTION_HEADER.read_text(), re.M)))


def test_binding_covers_the_header(lib):
    from consumer_int8 import _abi

    assert sorted(_abi.ATTENTION_SIGNATURES) == declared()
    for name in declared():
        assert hasattr(lib, name)


FAKE = 0x100000000  # never dereferenced


def heads(at=0, n=4, dim=128, token_stride=None, head_stride=None):
    from consumer_int8 import _abi as A

    return A.Heads(FAKE + at, n, n * dim if token_stride is None else token_stride,
                   dim if head_stride is None else head_stride)


def cache(dim=128, n=4, pages=8, page=16, at=FAKE << 8, **more):
    from consumer_int8 import _abi as A

    code, scale = n * page * dim // 2, n * page * dim // 32
    gap = 1 << 28
    c = A.Fp4CacheView(at, at + gap, at + 2 * gap, at + 3 * gap, code, scale, code, scale, pages, n, page)
    for name, value in more.items():
        setattr(c, name, value)
    return c


def rotation(**more):
    from consumer_int8 import _abi as A

    r = A.Rotation(FAKE << 4, 100, 64, FAKE << 5, 1, None, 0)
    for name, value in more.items():
        setattr(r, name, value)
    return r


def norm(**more):
    from consumer_int8 import _abi as A

    n = A.HeadNorm(FAKE << 6, FAKE << 6, 1e-6)
    for name, value in more.items():
        setattr(n, name, value)
    return n


def refused(lib, status, code, text):
    from consumer_int8 import _abi

    assert status == code, (status, _abi.last_error())
    assert text in _abi.last_error()


def codes():
    from consumer_int8 import _abi as A

    return A.CI8_ERR_GEOMETRY, A.CI8_ERR_ALIGNMENT, A.CI8_ERR_OVERLAP, A.CI8_ERR_TOO_LARGE


def test_qk_norm_rope_refusals(lib):
    geometry, alignment, overlap, large = codes()
    ref = ctypes.byref

    def call(q=None, k=None, q_out=None, k_out=None, n=None, r=None, tokens=8, dim=128):
        q, k = q or heads(), k or heads(1 << 24, 2)
        return lib.ci8_qk_norm_rope(ref(q), ref(k), ref(q_out or heads(1 << 25)),
                                    ref(k_out or heads(1 << 26, 2)), ref(n or norm()),
                                    ref(r or rotation()), tokens, dim, None)

    for dim in (0, 32, 96, 512):
        refused(lib, call(dim=dim), geometry, "Unsupported head size")
    refused(lib, call(tokens=-1), geometry, "Invalid token count")
    refused(lib, call(tokens=1 << 25), large, "Too many tokens")
    refused(lib, call(q=heads(n=0)), geometry, "Invalid heads")
    refused(lib, call(q=heads(token_stride=516)), alignment, "Heads require")
    refused(lib, call(k=heads((1 << 24) + 8, 2)), alignment, "Heads require")
    refused(lib, call(q=heads(token_stride=1 << 60)), large, "Heads too large")
    refused(lib, call(q_out=heads(1 << 25, 3)), geometry, "their inputs' heads")
    refused(lib, call(q_out=heads(1 << 25, head_stride=64)), overlap, "overlap each other")
    refused(lib, call(q_out=heads(1 << 25, token_stride=256)), overlap, "overlap each other")
    refused(lib, call(q_out=heads(64)), overlap, "An output must be its input")
    refused(lib, call(q_out=heads(1 << 24)), overlap, "An output must be its input")
    refused(lib, call(k_out=heads(1 << 25, 2)), overlap, "An output must be its input")
    refused(lib, call(n=norm(q_weight=(FAKE << 6) + 4)), alignment, "Norm weights")
    for eps in (-1.0, float("nan"), 1e60):
        refused(lib, call(n=norm(eps=eps)), geometry, "Invalid norm")
    for bad in [dict(rot=8), dict(rot=24), dict(rot=144), dict(rot=-16), dict(rows=0), dict(axes=0),
                dict(axes=3), dict(axes=17, axis_of=FAKE << 7), dict(table=None), dict(positions=None)]:
        refused(lib, call(r=rotation(**bad)), geometry, "Invalid rotation")
    refused(lib, call(r=rotation(table=(FAKE << 4) + 8)), alignment, "Rotation requires")
    refused(lib, call(q_out=heads((FAKE << 4) - FAKE)), overlap, "An output must be its input")


def test_views_of_one_buffer_are_told_apart(lib):
    """Heads of one projected row interleave without sharing an element. What passes every
    check has zero tokens here, so that nothing is launched."""
    geometry, alignment, overlap, large = codes()
    ref = ctypes.byref
    row = (4 + 2 + 2) * 128
    q, k = heads(0, 4, token_stride=row), heads(4 * 256, 2, token_stride=row)
    v = heads(6 * 256, 2, token_stride=row)

    def call(q_out, k_out, tokens):
        return lib.ci8_qk_norm_rope(ref(q), ref(k), ref(q_out), ref(k_out), ref(norm()), ref(rotation()),
                                    tokens, 128, None)

    assert call(q, k, 0) == 0
    # swapped in the row: each output lies on the other's input
    refused(lib, call(q, heads(0, 2, token_stride=row), 8), overlap, "An output must be its input")
    refused(lib, call(q, heads(3 * 256, 2, token_stride=row), 8), overlap, "An output must be its input")
    refused(lib, call(heads(5 * 256, 4, token_stride=row), k, 8), overlap, "An output must be its input")
    refused(lib, lib.ci8_append_fp4(ref(q), ref(k), ref(v), ref(heads(4 * 256, 4, token_stride=row)), ref(norm()),
                                    ref(rotation()), FAKE << 10, ref(cache(n=2)), 8, 128, None),
            overlap, "An output must be its input")


def test_append_and_unpack_refusals(lib):
    geometry, alignment, overlap, large = codes()
    ref = ctypes.byref

    def append(k=None, v=None, c=None, slots=FAKE << 10, tokens=8, dim=128, q=None, q_out=None):
        return lib.ci8_append_fp4(ref(q) if q else None, ref(k or heads()), ref(v or heads(1 << 24)),
                                  ref(q_out) if q_out else None, ref(norm()), ref(rotation()), slots,
                                  ref(c or cache()), tokens, dim, None)

    def unpack(c=None, slots=FAKE << 10, k=FAKE, v=FAKE + (1 << 24), count=8, dim=128):
        return lib.ci8_unpack_fp4(ref(c or cache()), slots, k, v, count, dim, None)

    for call in (append, unpack):
        for bad in [dict(pages=0), dict(page_size=8), dict(page_size=48), dict(page_size=2048), dict(heads=0)]:
            refused(lib, call(c=cache(**bad)), geometry, "Invalid cache")
        refused(lib, call(c=cache(k_code_page_stride=4 * 16 * 64 - 16)), geometry, "pages overlap")
        refused(lib, call(c=cache(at=(FAKE << 8) + 8)), alignment, "The cache requires")
        refused(lib, call(c=cache(v_scale_page_stride=4 * 16 * 4 + 4)), alignment, "The cache requires")
        refused(lib, call(c=cache(v_code_page_stride=1 << 46)), large, "Cache too large")
    refused(lib, append(k=heads(n=2)), geometry, "the cache's heads")
    refused(lib, append(slots=(FAKE << 10) + 4), alignment, "Slots")
    refused(lib, append(c=cache(v_codes=FAKE << 8)), overlap, "Cache buffers must not overlap")
    refused(lib, append(c=cache(v_scales=FAKE)), overlap, "The cache must not overlap an input")
    refused(lib, append(c=cache(v_scales=FAKE << 10)), overlap, "The cache must not overlap an input")
    refused(lib, append(q=heads(1 << 25), q_out=heads()), overlap, "An output must be its input")
    refused(lib, append(q=heads(1 << 25)), geometry, "Missing heads")
    refused(lib, unpack(k=FAKE + 8), alignment, "unpack_fp4 requires")
    refused(lib, unpack(v=FAKE + 64), overlap, "must not overlap")
    refused(lib, unpack(k=FAKE << 8), overlap, "must not overlap")
    refused(lib, unpack(count=-1), geometry, "Invalid token count")
    # keys and values of one pool: pages of four parts, strides the whole page
    page = 4 * 16 * (64 + 4) * 2
    at = FAKE << 8
    pool = cache(k_codes=at, v_codes=at + 4096, k_scales=at + 8192, v_scales=at + 8448,
                 **{n + "_page_stride": page for n in ("k_code", "k_scale", "v_code", "v_scale")})
    assert append(c=pool, tokens=0) == 0
    pool.v_scales = at + 8192 + 248
    refused(lib, append(c=pool), overlap, "Cache buffers must not overlap")


def test_attention_refusals(lib):
    geometry, alignment, overlap, large = codes()
    ref = ctypes.byref

    def call(q=None, c=None, table=FAKE << 10, width=4, lens=FAKE << 11, starts=None, seqs=8, tokens=8, dim=128,
             ws=FAKE << 12, out=FAKE + (1 << 26), lse=FAKE << 13, scale=0.1, max_q=1, window=0):
        return lib.ci8_attention_fp4(ref(q or heads(n=8)), ref(c or cache()), table, width, lens, starts, seqs,
                                     tokens, dim, ws, out, lse, scale, max_q, window, None)

    refused(lib, call(dim=80), geometry, "Unsupported head size")
    refused(lib, call(q=heads(n=6)), geometry, "a multiple of the cache's heads")
    for bad in [dict(seqs=-1), dict(seqs=1 << 17), dict(width=-1), dict(max_q=0), dict(window=-1),
                dict(scale=float("inf")), dict(scale=float("nan")), dict(seqs=4)]:
        refused(lib, call(**bad), geometry, "Invalid attention")
    refused(lib, call(width=1 << 28), large, "Page table too large")
    for bad in [dict(table=(FAKE << 10) + 2), dict(lens=(FAKE << 11) + 1), dict(ws=(FAKE << 12) + 8),
                dict(out=FAKE + (1 << 26) + 2), dict(lse=(FAKE << 13) + 2), dict(starts=(FAKE << 14) + 2)]:
        refused(lib, call(**bad), alignment, "attention_fp4 requires aligned")
    for bad in [dict(out=FAKE), dict(out=FAKE << 8), dict(lse=FAKE + (1 << 26)), dict(ws=FAKE << 10),
                dict(lse=FAKE << 11), dict(out=(FAKE << 12) + 64)]:
        refused(lib, call(**bad), overlap, "must not overlap anything else")
    assert call(seqs=0, tokens=0) == 0 and call(seqs=3, tokens=0, starts=FAKE << 14) == 0


def test_schemas_and_fakes():
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode

    from consumer_int8 import attention

    assert "Tensor(a!)? q_out" in str(attention.append_fp4.default._schema)
    with FakeTensorMode():
        q = torch.empty(2, 4, 64, dtype=torch.bfloat16)
        k = torch.empty(2, 2, 64, dtype=torch.bfloat16)
        at = torch.empty(2, dtype=torch.int64)
        c = attention.new_cache(4, 2, 16, 64, device="cpu")
        assert attention.qk_norm_rope(q, k, None, None, None, None, None, q, k) is None
        assert attention.append_fp4(q, k, k, None, None, None, None, None, at, q, *c) is None
        assert attention.unpack_fp4(*c, at, k, k) is None
        i32 = torch.empty(2, dtype=torch.int32)
        assert attention.attention_fp4(q, *c, torch.empty(2, 3, dtype=torch.int32), i32, None,
                                       torch.empty(66, 4), torch.empty_like(q), None, 0.1) is None


def test_no_cpu_implementation():
    import torch

    from consumer_int8 import attention

    k = torch.empty(2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        attention.unpack_fp4(*attention.new_cache(4, 2, 16, 64, device="cpu"), torch.empty(2, dtype=torch.int64), k, k)


def test_rope_table():
    import torch

    from consumer_int8 import attention

    t = attention.rope_table(7, 32, 500.0, device="cpu")
    angle = np.arange(7)[:, None] * 500.0 ** (-np.arange(16) / 16)
    assert t.shape == (7, 32) and t.dtype == torch.float32
    assert np.allclose(t.numpy(), np.concatenate([np.cos(angle), np.sin(angle)], 1), atol=1e-6)
    with pytest.raises(ValueError):
        attention.rope_table(7, 24)
    with pytest.raises(ValueError):
        attention.new_cache(1, 1, 16, 96, device="cpu")


def test_extent_refusals(lib):
    """What the kernels hold in 32 bits: places of pages, and sums of the tiles of 64 sequences."""
    *_, large = codes()
    ref = ctypes.byref

    def call(c, width):
        return lib.ci8_attention_fp4(ref(heads(n=8)), ref(c), FAKE << 10, width, FAKE << 11, None, 0, 0, 128,
                                     FAKE << 12, FAKE + (1 << 26), None, 0.1, 1, 0, None)

    size = cache().page_size
    most = ((1 << 26) - 4096) // size
    refused(lib, call(cache(), most + 1), large, "Page table too large")
    assert call(cache(), most) == 0
    far = dict(k_codes=1 << 40, k_scales=1 << 41, v_codes=1 << 42, v_scales=1 << 43)
    for name in far:
        stride = {name[:-1] + "_page_stride": 1 << 33}
        refused(lib, call(cache(pages=5, **far, **stride), 4), large, "Cache too large")
        assert call(cache(pages=4, **far, **stride), 4) == 0
