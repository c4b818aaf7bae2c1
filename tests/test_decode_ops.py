"""CPU: refusals of the operators around the delta, through the C ABI and through Python (tensors without storage), and
the oracle's own consistency."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import decode_oracle as O


def test_abi_refusals(lib):
    from ae296_b200._lib import Append, Attention, Int4, KvCache
    p = 1 << 20
    cache = KvCache(p, p, 16 * 2 * 128, 2 * 128, 128, 10, 16, 2, 128)

    def append(c=cache, dtype=0, **kw):
        a = Append()
        for n in ("q_out", "q", "k", "v", "positions", "slots", "cos", "sin"):
            setattr(a, n, p)
        a.n_positions, a.rotary_dim, a.n_tokens, a.n_heads = 64, 128, 4, 8
        for n, v in kw.items():
            setattr(a, n, v)
        return lib.b200_kv_append(C.byref(a), C.byref(c) if c else None, dtype, None)

    assert append(c=None) == -1 and append(q=None) == -1 and append(slots=None) == -1 and append(cos=None) == -1
    assert append(dtype=2) == -3
    for kw in (dict(rotary_dim=130), dict(rotary_dim=3), dict(rotary_dim=0), dict(n_tokens=-1), dict(n_heads=0), dict(n_positions=0),
               dict(c=KvCache(p, p, 0, 0, 0, 10, 16, 2, 514)), dict(c=KvCache(p, p, 0, 0, 0, 0, 16, 2, 128)), dict(c=KvCache(p, p, 0, 0, 0, 10, 16, 2, 127))):
        assert append(**kw) == -2, kw
    assert append(n_tokens=0) == 0
    assert lib.b200_kv_append(None, C.byref(cache), 0, None) == -1

    need = lib.b200_prefix_attention_workspace_bytes(4, 1, 8, 2, 128)

    def attend(c=cache, dtype=0, workspace=p, nbytes=need, **kw):
        a = Attention()
        for n in ("out", "q", "table", "lens", "prefix_table", "prefix_lens", "group_starts"):
            setattr(a, n, p)
        a.max_pages, a.max_prefix_pages, a.n_requests, a.n_groups, a.n_heads, a.scale = 3, 3, 4, 1, 8, 1.0
        for n, v in kw.items():
            setattr(a, n, v)
        return lib.b200_prefix_attention(C.byref(a), C.byref(c) if c else None, dtype, workspace, nbytes, None)

    for kw in (dict(c=None), dict(out=None), dict(q=None), dict(lens=None), dict(table=None), dict(prefix_table=None), dict(prefix_lens=None),
               dict(group_starts=None), dict(workspace=None)):
        assert attend(**kw) == -1, kw
    assert attend(dtype=2) == -3
    for kw in (dict(n_heads=7), dict(n_heads=0), dict(n_heads=1026), dict(n_requests=4097), dict(n_requests=-1), dict(n_groups=2049), dict(n_groups=-1),
               dict(max_pages=-1), dict(max_pages=1 << 28), dict(max_prefix_pages=1 << 28), dict(c=KvCache(p, p, 0, 0, 0, 10, 24, 2, 128)),
               dict(c=KvCache(p, p, 0, 0, 0, 10, 512, 2, 128)), dict(c=KvCache(p, p, 0, 0, 0, 10, 16, 2, 96)), dict(c=KvCache(p, p, 0, 0, 0, 10, 0, 2, 128))):
        assert attend(**kw) == -2, kw
    for kw in (dict(q=p + 2), dict(out=p + 8), dict(workspace=p + 4), dict(q_row=4), dict(out_head=2), dict(c=KvCache(p + 2, p, 0, 0, 0, 10, 16, 2, 128)),
               dict(c=KvCache(p, p, 0, 0, 4, 10, 16, 2, 128))):
        assert attend(**kw) == -4, kw
    assert attend(nbytes=need - 1) == -6
    assert attend(n_requests=0) == 0
    size = lib.b200_prefix_attention_workspace_bytes
    assert size(0, 0, 8, 2, 128) == size(4, 0, 9, 2, 128) == size(4, 0, 8, 2, 80) == 0 and size(4, 0, 8, 2, 64) > 0
    assert size(4096, 1, 64, 8, 128) < 2 ** 30                  # one group of a large batch needs no more than its tiles

    def int4(dtype=0, y_dtype=0, **kw):
        a = Int4()
        for n in ("y", "x", "codes", "scales"):
            setattr(a, n, p)
        a.x_row, a.y_row, a.n_tokens, a.n_in, a.n_out, a.group = 256, 64, 2, 256, 64, 64
        for n, v in kw.items():
            setattr(a, n, v)
        return lib.b200_int4_linear(C.byref(a), dtype, y_dtype, None)

    assert int4(y=None) == int4(x=None) == int4(codes=None) == int4(scales=None) == -1
    assert int4(dtype=2) == int4(y_dtype=1) == int4(dtype=1, y_dtype=0) == -3
    for kw in (dict(group=16), dict(group=256), dict(n_in=224), dict(n_in=0), dict(n_out=0), dict(n_tokens=-1), dict(n_tokens=65535 * 32 + 1), dict(x_row=248)):
        assert int4(**kw) == -2, kw
    assert int4(x=p + 2) == int4(codes=p + 8) == int4(x_row=260) == -4
    assert int4(n_tokens=0) == 0


def fake(*shape, dtype=torch.float16):
    """A CUDA tensor without storage, on any machine."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(allow_non_fake_inputs=True):
        return torch.empty(*shape, dtype=dtype, device="cuda")


I32, I64, F32, BF = torch.int32, torch.int64, torch.float32, torch.bfloat16


def test_python_refusals_of_append(lib):
    import ae296_b200 as L
    good = dict(q_out=fake(4, 8, 64), q=fake(4, 8, 64), k=fake(4, 2, 64), v=fake(4, 2, 64), k_cache=fake(5, 16, 2, 64), v_cache=fake(5, 16, 2, 64),
                positions=fake(4, dtype=I64), slots=fake(4, dtype=I32), cos=fake(9, 32, dtype=F32), sin=fake(9, 32, dtype=F32))
    bad = [dict(q=fake(4, 8, 32)), dict(q=fake(4, 512)), dict(q_out=fake(3, 8, 64)), dict(k=fake(4, 3, 64)), dict(v=fake(4, 2, 64, dtype=BF)),
           dict(k_cache=fake(5, 16, 2, 64, dtype=BF)), dict(v_cache=fake(6, 16, 2, 64)), dict(v_cache=fake(5, 2, 16, 64).transpose(1, 2)),
           dict(k_cache=fake(0, 16, 2, 64), v_cache=fake(0, 16, 2, 64)), dict(positions=fake(5, dtype=I64)), dict(slots=fake(4, dtype=torch.int16)),
           dict(slots=fake(8, dtype=I32)[::2]), dict(cos=fake(9, 33, dtype=F32), sin=fake(9, 33, dtype=F32)), dict(sin=fake(8, 32, dtype=F32)),
           dict(cos=fake(9, 32, dtype=BF), sin=fake(9, 32, dtype=BF)), dict(cos=fake(0, 32, dtype=F32), sin=fake(0, 32, dtype=F32)),
           dict(dq=fake(4, 8, 63)), dict(dk=fake(4, 2, 64, dtype=F32)), dict(dv=fake(4, 64, 2).transpose(1, 2)), dict(q=fake(4, 64, 8).transpose(1, 2)),
           dict(status=fake(1, dtype=I64)), dict(status=fake(2, dtype=I32)), dict(q=torch.empty(4, 8, 64, dtype=torch.float16)), dict(k=None), dict(q=fake(4, 8, 64, dtype=F32))]
    for kw in bad:
        with pytest.raises(ValueError):
            L.append_kv(**dict(good, **kw))


def test_python_refusals_of_attention(lib):
    import ae296_b200 as L
    good = dict(out=fake(4, 8, 64), q=fake(4, 8, 64), k_cache=fake(5, 16, 2, 64), v_cache=fake(5, 16, 2, 64), block_table=fake(4, 3, dtype=I32),
                lens=fake(4, dtype=I32))
    pre = dict(prefix_table=fake(2, 3, dtype=I32), prefix_lens=fake(2, dtype=I32), group_starts=fake(3, dtype=I32))
    bad = [dict(out=fake(4, 8, 64, dtype=BF)), dict(out=fake(4, 9, 64)), dict(q=fake(4, 7, 64), out=fake(4, 7, 64)), dict(lens=fake(4, dtype=I64)),
           dict(lens=fake(3, dtype=I32)), dict(block_table=fake(3, 3, dtype=I32)), dict(block_table=fake(4, 3, dtype=I64)), dict(block_table=fake(3, 4, dtype=I32).t()),
           dict(k_cache=fake(5, 16, 2, 32), v_cache=fake(5, 16, 2, 32)), dict(v_cache=fake(5, 16, 2, 64, dtype=BF)), dict(lse=fake(4, 8)),
           dict(lse=fake(8, 4, dtype=F32).t()), dict(pre, prefix_lens=None), dict(pre, group_starts=fake(2, dtype=I32)), dict(pre, prefix_lens=fake(3, dtype=I32)),
           dict(pre, prefix_table=fake(2, 3, dtype=I64)), dict(status=fake(1)), dict(q=torch.empty(4, 8, 64, dtype=torch.float16))]
    for kw in bad:
        with pytest.raises(ValueError):
            L.prefix_attention(**dict(good, **kw))
    wide = dict(good, out=fake(4097, 8, 64), q=fake(4097, 8, 64), block_table=fake(4097, 3, dtype=I32), lens=fake(4097, dtype=I32))
    many = dict(good, prefix_table=fake(2049, 3, dtype=I32), prefix_lens=fake(2049, dtype=I32), group_starts=fake(2050, dtype=I32))
    for kw in (wide, many):
        with pytest.raises((ValueError, RuntimeError)):
            L.prefix_attention(**kw)


def test_python_refusals_of_int4(lib):
    import ae296_b200 as L
    U8 = torch.uint8
    good = dict(y=fake(3, 40), x=fake(3, 256), codes=fake(40, 128, dtype=U8), scales=fake(40, 4))
    bad = [dict(y=fake(3, 41)), dict(y=fake(3, 40, dtype=BF)), dict(x=fake(3, 256, dtype=F32)), dict(codes=fake(40, 256, dtype=U8)), dict(codes=fake(40, 128)),
           dict(codes=fake(128, 40, dtype=U8).t()), dict(scales=fake(40, 3)), dict(scales=fake(40, 16)), dict(scales=fake(40, 1)), dict(scales=fake(40, 4, dtype=BF)),
           dict(scales=fake(4, 40).t()), dict(zeros=fake(40, 3, dtype=U8)), dict(zeros=fake(40, 4)), dict(add=fake(3, 40, dtype=F32)), dict(add=fake(2, 40)),
           dict(x=fake(256, 3).t()), dict(y=fake(40, 3).t()), dict(x=torch.empty(3, 256, dtype=torch.float16))]
    for kw in bad:
        with pytest.raises(ValueError):
            L.int4_linear(**dict(good, **kw))


def test_unreadable_tensors_raise(lib):
    """Operands in order but without storage: the exception of the same access in Python, no crash."""
    import ae296_b200 as L
    with pytest.raises(Exception):
        L.int4_linear(fake(3, 40), fake(3, 256), fake(40, 128, dtype=torch.uint8), fake(40, 4))
    with pytest.raises(Exception):
        L.prefix_attention(fake(4, 8, 64), fake(4, 8, 64), fake(5, 16, 2, 64), fake(5, 16, 2, 64), fake(4, 3, dtype=I32), fake(4, dtype=I32))


def test_oracle_identities():
    rng = np.random.default_rng(0)
    x, a = rng.normal(size=(3, 8)), rng.normal(size=(3, 4))
    for inter in (False, True):
        y = O.rotate(x, np.cos(a), np.sin(a), 8, inter)
        np.testing.assert_allclose((y ** 2).sum(-1), (x ** 2).sum(-1))                       # a rotation keeps lengths
        np.testing.assert_allclose(O.rotate(y, np.cos(a), -np.sin(a), 8, inter), x)          # and is undone by its inverse
    q, kc, vc = rng.normal(size=(3, 4, 8)), rng.normal(size=(6, 4, 2, 8)), rng.normal(size=(6, 4, 2, 8))
    table, pre = np.array([[0, 1], [2, 3], [4, 0]]), np.array([[5, 1]])
    whole = O.attention(q, kc, vc, np.concatenate([np.repeat(pre, 3, 0)[:, :1], table], 1), [4 + 7, 4 + 3, 4 + 1])
    split = O.attention(q, kc, vc, table, [7, 3, 1], pre, [4], [0, 3])
    for w, s in zip(whole, split):                                                           # a prefix of whole pages is a longer table
        np.testing.assert_allclose(w, s)
    codes = np.array([[0x21, 0xF0]], np.uint8)
    np.testing.assert_array_equal(O.int4_weights(codes, np.array([[2.0]])), [[-14.0, -12.0, -16.0, 14.0]])


def test_int4_refuses_sizes_that_do_not_round_up_in_32_bits(lib):
    from ae296_b200._lib import Int4
    for kw in (dict(n_in=2 ** 31 - 128), dict(n_in=2 ** 31 - 32, group=32), dict(n_out=2 ** 31 - 255), dict(n_out=2 ** 31 - 1), dict(n_out=2 ** 31 - 1, n_tokens=40)):
        a = Int4()
        a.y = a.x = a.codes = a.scales = 1 << 20
        a.x_row, a.y_row, a.n_tokens, a.n_in, a.n_out, a.group = 2 ** 31, 2 ** 31, 2, 256, 64, 64
        for n, v in kw.items():
            setattr(a, n, v)
        assert lib.b200_int4_linear(C.byref(a), 0, 0, None) == -2, kw


def test_int4_takes_a_status_word_and_refuses_others(lib):
    import ae296_b200 as L
    good = dict(y=fake(3, 40), x=fake(3, 256), codes=fake(40, 128, dtype=torch.uint8), scales=fake(40, 4))
    for word in (fake(1, dtype=I64), fake(2, dtype=I32), fake(1, dtype=F32), torch.zeros(1, dtype=I32)):
        with pytest.raises(ValueError):
            L.int4_linear(**good, status=word)


def test_attention_names_what_is_wrong_with_odd_arguments(lib):
    """What has no shape, or not the dimensions that the default scale and the number of groups are read from."""
    import ae296_b200 as L
    good = dict(out=fake(4, 8, 64), q=fake(4, 8, 64), k_cache=fake(5, 16, 2, 64), v_cache=fake(5, 16, 2, 64), block_table=fake(4, 3, dtype=I32), lens=fake(4, dtype=I32))
    pre = dict(prefix_table=fake(2, 3, dtype=I32), prefix_lens=fake(2, dtype=I32), group_starts=fake(3, dtype=I32))
    for kw, why in ((dict(q=None), "tensors expected"), (dict(q=[1.0]), "tensors expected"), (dict(q=fake(()), out=fake(())), "q must be"),
                    (dict(q=fake(4, 8, 0), out=fake(4, 8, 0)), "head_dim"), (dict(pre, prefix_table=fake((), dtype=I32)), "groups"),
                    (dict(pre, prefix_table=fake(2, dtype=I32)), "groups"), (dict(scale="0.1"), "number")):
        with pytest.raises(ValueError, match=why):
            L.prefix_attention(**dict(good, **kw))


def test_structures_have_the_header_s_sizes(tmp_path):
    """The ctypes structures against the C compiler's."""
    import os
    import shutil
    import subprocess
    from ae296_b200 import _lib
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    pairs = [("b200_kv_cache", _lib.KvCache), ("b200_append", _lib.Append), ("b200_attention", _lib.Attention), ("b200_int4", _lib.Int4)]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "b200_decode.h"\nint main(void) {\n' + "".join(
        f'    printf("%zu\\n", sizeof({c}));\n' + "".join(f'    printf("%zu\\n", offsetof({c}, {n}));\n' for n, _ in t._fields_) for c, t in pairs) + "    return 0;\n}\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run([cc, "-I", include, str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [x for _, t in pairs for x in (C.sizeof(t), *(getattr(t, n).offset for n, _ in t._fields_))]
