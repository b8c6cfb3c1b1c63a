"""CPU tests of the text decoder's C entry points: declared symbols, sizes,
and what they refuse before anything reaches a GPU."""

import ctypes

import pytest

from test_cpu_abi import declared, exported


def test_library_exports_decode_entry_points():
    from ppocr_b200 import capi

    names = declared("ppocr_b200_decode.h")
    assert len(set(names)) == 6
    assert set(names) <= exported(capi.lib_path()) and set(names) <= set(capi.SIGNATURES)


@pytest.mark.parametrize("page,dim,want", [(16, 32, 640), (32, 64, 2560), (64, 128, 10240), (128, 128, 20480),
                                           (0, 64, 0), (48, 64, 0), (256, 64, 0), (32, 96, 0), (32, 0, 0)])
def test_block_bytes(page, dim, want):
    from oracle import decode as O
    from ppocr_b200 import capi

    assert capi.load().ppocr_b200_kv4_block_bytes(page, dim) == want
    if want:
        assert O.block_bytes(page, dim) == want


def geometry(**kw):
    from ppocr_b200 import capi

    g = dict(pool=0x1000, pages=8, page_size=32, kv_heads=2, head_dim=64, type=0) | kw
    return ctypes.byref(capi.PpocrKv4Cache(*g.values()))


PLACES = dict(table=0x2000, width=4, lengths=0x3000, starts=0x4000, batch=2, tokens=3, max_new=2)


@pytest.mark.parametrize("cache,places,what", [
    (dict(pool=None), {}, "pool"),
    (dict(pool=0x1008), {}, "pool"),
    (dict(type=2), {}, "type"),
    (dict(page_size=48), {}, "page size"),
    (dict(head_dim=96), {}, "head_dim"),
    (dict(kv_heads=0), {}, "kv_heads"),
    (dict(kv_heads=4097), {}, "kv_heads"),
    (dict(pages=1 << 31), {}, "2^31"),
    ({}, dict(table=None), "table"),
    ({}, dict(lengths=None), "lengths"),
    ({}, dict(width=0), "width"),
    ({}, dict(width=1 << 27), "width"),
    ({}, dict(batch=-1), "batch"),
    ({}, dict(batch=65536), "batch"),
    ({}, dict(tokens=-1), "tokens"),
    ({}, dict(starts=None), "batch * max_new"),
])
def test_cache_calls_refuse(cache, places, what):
    from ppocr_b200 import capi

    lib = capi.load()
    c = geometry(**cache)
    p = list((PLACES | places).values())
    assert lib.ppocr_b200_kv4_append(c, 0x5000, 128, 0x6000, 128, *p, None) == -1
    assert what in lib.ppocr_b200_last_error().decode()
    assert lib.ppocr_b200_kv4_read(c, 0x5000, 0x6000, *p, None) == -1
    assert what in lib.ppocr_b200_last_error().decode()
    assert lib.ppocr_b200_kv4_attention(c, 0x5000, 256, 0x6000, 4, 0.125, 0, 0, *p, 0x10000, None) == -1
    assert what in lib.ppocr_b200_last_error().decode()


def test_null_cache():
    from ppocr_b200 import capi

    lib = capi.load()
    assert lib.ppocr_b200_kv4_append(None, 0x5000, 128, 0x6000, 128, *PLACES.values(), None) == -1


def test_row_arguments():
    from ppocr_b200 import capi

    lib = capi.load()
    c, p = geometry(), list(PLACES.values())
    append = [(0x5008, 128, 0x6000, 128), (0x5000, 120, 0x6000, 128), (0x5000, 132, 0x6000, 128),
              (None, 128, 0x6000, 128), (0x5000, 128, 0x6000, 64)]
    for args in append:
        assert lib.ppocr_b200_kv4_append(c, *args, *p, None) == -1, args
    assert lib.ppocr_b200_kv4_read(c, None, 0x6000, *p, None) == -1
    good = dict(q=0x5000, stride=256, out=0x6000, heads=4, scale=0.125, window=0, sinks=0)
    for bad in (dict(q=0x5002), dict(q=None), dict(out=0x6008), dict(stride=248), dict(stride=260), dict(heads=3),
                dict(heads=0), dict(heads=65538, stride=65538 * 64), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(sinks=-2)):
        assert lib.ppocr_b200_kv4_attention(c, *(good | bad).values(), *p, 0x10000, None) == -1, bad
    for workspace in (None, 0x10080):
        assert lib.ppocr_b200_kv4_attention(c, *good.values(), *p, workspace, None) == -1
        assert "workspace" in lib.ppocr_b200_last_error().decode()


def test_empty_calls_do_nothing():
    from ppocr_b200 import capi

    lib = capi.load()
    c = geometry()
    for places in (dict(batch=0, tokens=0), dict(tokens=0), dict(max_new=0)):
        p = list((PLACES | places).values())
        assert lib.ppocr_b200_kv4_append(c, None, 128, None, 128, *p, None) == 0
        assert lib.ppocr_b200_kv4_read(c, None, None, *p, None) == 0
        assert lib.ppocr_b200_kv4_attention(c, None, 256, None, 4, 0.125, 0, 0, *p, None, None) == 0
    assert lib.ppocr_b200_sample(None, 0, 10, 0, 10, None, None, None, None, None, None, None, None, None) == 0


def test_sample_refuses():
    from ppocr_b200 import capi

    lib = capi.load()
    good = dict(logits=0x1000, type=0, stride=100, rows=4, vocab=100, t=None, k=None, p=None, m=None, u=0x2000,
                ids=0x3000, prob=0x4000, kept=0x5000)
    for bad in (dict(logits=None), dict(logits=0x1001), dict(type=3), dict(type=2, logits=0x1002), dict(stride=99),
                dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 24) + 1, stride=1 << 25), dict(u=None), dict(ids=None),
                dict(prob=None), dict(kept=None)):
        assert lib.ppocr_b200_sample(*(good | bad).values(), None) == -1, bad
        assert lib.ppocr_b200_last_error().decode().startswith("sample: ")


def test_python_front_refuses():
    """decode.KvCache4 and decode.sample name the argument."""
    import torch

    from ppocr_b200 import decode

    with pytest.raises(ValueError, match="dtype"):
        decode.KvCache4(4, 16, 2, 64, dtype=torch.float32, device="cpu")
    with pytest.raises(ValueError, match="page_size"):
        decode.KvCache4(4, 24, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="pool"):
        decode.KvCache4(4, 16, 2, 64, device="cpu", pool=torch.zeros(4, 2, 100, dtype=torch.uint8))
    c = decode.KvCache4(4, 16, 2, 64, device="cpu")
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    k = torch.zeros(2, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="k must be"):
        c.append(k.float(), k, table, lens)
    with pytest.raises(ValueError, match="side by side"):
        c.append(torch.zeros(2, 2, 128, dtype=torch.float16)[..., :64], k, table, lens)
    with pytest.raises(ValueError, match="table"):
        c.append(k, k, table.long(), lens)
    with pytest.raises(ValueError, match="lengths"):
        c.append(k, k, table, lens[:1])
    with pytest.raises(ValueError, match="divide"):
        c.append(k[:1], k[:1], table, lens)
    with pytest.raises(ValueError, match="max_new"):
        c.append(k, k, table, lens, starts=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="out"):
        c.attention(k, table, lens, out=torch.zeros(2, 2, 64))
    with pytest.raises(ValueError, match="logits"):
        decode.sample(torch.zeros(2, 10), torch.zeros(2))


def test_quantised_values_stay_within_half_a_step():
    """The format itself, on the restatement the kernels are held to."""
    import torch

    from oracle import decode as O

    g = torch.Generator().manual_seed(1)
    for t in (torch.float16, torch.bfloat16):
        x = (torch.randn(50, 3, 96, generator=g) * 3).to(t)
        codes, scale, low = O.quantise(x)
        y = O.restore(codes, scale, low)
        u = 2.0 ** -11 if t == torch.float16 else 2.0 ** -8
        step = scale.double().repeat_interleave(32, -1)
        assert ((y - x.double()).abs() <= step * (0.5 + 16 * u) + 1e-6).all()
        assert int(codes.max()) == 15 and int(codes.min()) == 0
