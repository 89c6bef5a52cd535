"""Refusals of the paged-cache entries, checked on the host (no device needed):
every bad argument comes back as a PJRT error code with a message before any CUDA call."""
import ctypes
import os
import subprocess

import pytest

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def paged():
    import __graft_entry__
    __graft_entry__.build()
    from cljxla_b200.host import paged as m
    return m


def cache(paged, **kw):
    c = paged._Cache(ctypes.sizeof(paged._Cache), 0x10000, 0x20000, 4096, 1024, 64, 4096, 1024, 64, 8, 4, 16, 64,
                     0x30000, 0x40000, 2, 5, 5, paged.DTYPE_ENUM["bf16"], 0)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def append_args(paged, **kw):
    a = paged._AppendArgs(ctypes.sizeof(paged._AppendArgs), 0x50000, 0x60000, 0x70000, 0x80000, 4, 8, 256, 64, 256, 64, 512,
                          64, 512, 64, None, 0x90000, 64, 0, 1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def attention_args(paged, **kw):
    a = paged._AttentionArgs(ctypes.sizeof(paged._AttentionArgs), 0x50000, 0x60000, 4, 8, 512, 64, 512, 64, None, 2, -1, 0.125,
                             0.0, paged.DTYPE_ENUM["bf16"], 0, None, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def verify_args(paged, **kw):
    a = paged._VerifyArgs(ctypes.sizeof(paged._VerifyArgs), 0x10000, 0x20000, 0x30000, None, 0x40000, 0x50000, 4, 2, 100, 2,
                          100, 100, 100, 1.0, 1.0, paged.DTYPE_ENUM["bf16"], 0, 0x60000, 0x70000, 0x80000, 0x90000, 0xa0000,
                          None, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def call(f, *structs):
    err = ctypes.create_string_buffer(512)
    rc = f(*[None if s is None else ctypes.addressof(s) for s in structs], None, err, 512)
    return rc, err.value.decode()


CACHE_BAD = [
    (dict(struct_size=8), "struct_size"), (dict(head_dim=96), "head_dim"), (dict(head_dim=0), "head_dim"),
    (dict(kv_heads=0), "kv_heads"), (dict(page_size=0), "page_size"), (dict(num_pages=-1), "num_pages"),
    (dict(num_pages=1 << 31), "num_pages"), (dict(num_seqs=-1), "num_seqs"), (dict(pages_per_seq=-1), "pages_per_seq"),
    (dict(pages_per_seq=1 << 27, page_table_stride=1 << 27), "2^30"), (dict(page_table_stride=4), "page_table"),
    (dict(k_page_stride=-1), "k_page_stride"), (dict(v_row_stride=1 << 50), "v_row_stride"),
    (dict(k_row_stride=65), "16-byte"), (dict(v_head_stride=1025), "16-byte"), (dict(k_pages=0x10002), "16-byte"),
    (dict(dtype=4), "dtype"), (dict(seq_lens=None), "seq_lens"), (dict(page_table=None), "page_table"),
    (dict(v_pages=None), "null pages"),
]


@pytest.mark.parametrize("kw,msg", CACHE_BAD)
def test_cache_refusals(paged, kw, msg):
    lib = paged._library()
    for f, a in ((lib.append, append_args(paged)), (lib.attend, attention_args(paged))):
        rc, err = call(f, cache(paged, **kw), a)
        assert rc == 3 and msg in err, (rc, err)


@pytest.mark.parametrize("kw,msg", [
    (dict(struct_size=8), "struct_size"), (dict(rotary_dim=65), "rotary_dim"), (dict(rotary_dim=66), "rotary_dim"),
    (dict(rotary_dim=-2), "rotary_dim"), (dict(inv_freq=None), "inv_freq"), (dict(q_out=None), "q_out"),
    (dict(q=None), "q_out"), (dict(q_heads=0), "q_heads"), (dict(tokens=3), "multiple of num_seqs"),
    (dict(tokens=-1), "tokens"), (dict(k=None), "null k"), (dict(v_token_stride=-1), "v_token_stride"),
    (dict(q_out_head_stride=0), "broadcast"), (dict(rope_scale=float("nan")), "rope_scale"),
    (dict(rope_scale=float("inf")), "rope_scale"),
    (dict(q_out=0x70000, q_out_head_stride=128, q_out_token_stride=1024), "strides of q"),
])
def test_append_refusals(paged, kw, msg):
    rc, err = call(paged._library().append, cache(paged), append_args(paged, **kw))
    assert rc == 3 and msg in err, (rc, err)


def test_append_refuses_broadcast_pages(paged):
    rc, err = call(paged._library().append, cache(paged, k_head_stride=0), append_args(paged))
    assert rc == 3 and "broadcast" in err


@pytest.mark.parametrize("kw,msg", [
    (dict(struct_size=8), "struct_size"), (dict(q_heads=6), "multiple of kv_heads"), (dict(q_heads=0), "q_heads"),
    (dict(tokens=3), "multiple of num_seqs"), (dict(max_tokens=1), "max_tokens"), (dict(max_tokens=-1), "max_tokens"),
    (dict(out_dtype=10), "out_dtype"), (dict(out_dtype=2), "dtype"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("inf")), "softcap"),
    (dict(scale=1e30, softcap=1e-30), "scale / softcap"), (dict(q=0x50008), "q must"), (dict(out=0x60004), "out must"), (dict(q_head_stride=65), "q must"),
    (dict(out_token_stride=0), "broadcast"), (dict(q=None), "null q"), (dict(out=None), "null q or out"),
    (dict(workspace=0x1008, workspace_bytes=1 << 40), "workspace"),
])
def test_attention_refusals(paged, kw, msg):
    rc, err = call(paged._library().attend, cache(paged), attention_args(paged, **kw))
    assert rc == 3 and msg in err, (rc, err)


@pytest.mark.parametrize("kw,msg", [
    (dict(struct_size=8), "struct_size"), (dict(vocab=0), "vocab"), (dict(max_tokens=0), "max_tokens"),
    (dict(max_tokens=129), "max_tokens"), (dict(max_tokens=1), "max_tokens"), (dict(tokens=3), "multiple of num_seqs"),
    (dict(target_stride=99), "target rows"), (dict(draft_stride=99), "draft rows"), (dict(race_stride=99), "race rows"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(temperature=4e-39), "temperature"), (dict(draft_temperature=-1.0), "draft_temperature"),
    (dict(dtype=4), "dtype"), (dict(tokens_out=None), "tokens_out"), (dict(accepted=None), "accepted"),
    (dict(seq_lens=None), "seq_lens"), (dict(target=None), "null target"), (dict(tokens_in=None), "tokens_in"),
    (dict(uniform=None), "uniform"), (dict(race=None), "race"), (dict(target=0x10001), "aligned"),
    (dict(num_seqs=-1), "num_seqs"), (dict(tokens=1 << 25), "tokens"),
])
def test_verify_refusals(paged, kw, msg):
    rc, err = call(paged._library().verify, verify_args(paged, **kw))
    assert rc == 3 and msg in err, (rc, err)


def test_null_structs_are_refused(paged):
    lib = paged._library()
    rc, err = call(lib.append, None, append_args(paged))
    assert rc == 3 and "null cache" in err
    for f, n in ((lib.append, 2), (lib.attend, 2), (lib.verify, 1)):
        rc, err = call(f, *([cache(paged)] if n == 2 else []), None)
        assert rc == 3 and "null arguments" in err
    # no message buffer: the code still comes back
    a = verify_args(paged, vocab=0)
    assert lib.verify(ctypes.addressof(a), None, None, 0) == 3


def test_nothing_to_do_succeeds_without_a_device(paged):
    lib = paged._library()
    assert call(lib.append, cache(paged), append_args(paged, tokens=0))[0] == 0
    assert call(lib.attend, cache(paged), attention_args(paged, tokens=0))[0] == 0
    assert call(lib.append, cache(paged, num_seqs=0), append_args(paged))[0] == 0
    assert call(lib.verify, verify_args(paged, num_seqs=0, tokens=0))[0] == 0


def test_struct_layouts_match_the_header(paged, tmp_path):
    """The ctypes mirrors have the header's sizes and offsets."""
    pairs = {"CLJXLA_PagedKV": paged._Cache, "CLJXLA_PagedAppendArgs": paged._AppendArgs,
             "CLJXLA_PagedAttentionArgs": paged._AttentionArgs, "CLJXLA_VerifyDraftArgs": paged._VerifyArgs}
    src = "#include <stdio.h>\n#include \"cljxla_b200.h\"\nint main(void) {\n"
    want = []
    for c, t in pairs.items():
        src += f'printf("%zu\\n", sizeof({c}));\n'
        want.append(ctypes.sizeof(t))
        for f, _ in t._fields_:
            src += f'printf("%zu\\n", offsetof({c}, {f}));\n'
            want.append(getattr(t, f).offset)
    (tmp_path / "l.c").write_text(src + "return 0; }\n")
    subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    assert [s.size for s in (paged._APPEND, paged._ATTENTION, paged._VERIFY)] == \
        [ctypes.sizeof(t) for t in (paged._AppendArgs, paged._AttentionArgs, paged._VerifyArgs)]
    got = subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == want


def test_python_refuses_host_tensors_and_bad_shapes(paged):
    z = torch.zeros
    with pytest.raises(ValueError, match="k_pages"):
        paged.PagedKV(z(2, 1, 16, 64), z(2, 1, 16, 64), z(1, 2, dtype=torch.int32), z(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="target_logits"):
        paged.verify_draft(z(2, 9), z(2, dtype=torch.int32), out_tokens=z(1, 2, dtype=torch.int32), accepted=z(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="inv_freq"):
        paged.Rope(z(4))


def test_rope_frequencies(paged):
    f = paged.rope_inv_freq(8, 100.0)
    assert torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75]))
    assert torch.allclose(paged.rope_inv_freq(8, 100.0, factor=4.0), f / 4)
    assert paged.rope_inv_freq(8, 100.0, proportion=0.5).tolist()[2:] == [0.0, 0.0]
    # 1000 trained positions: 159, 50, 16 and 5 turns
    g = paged.rope_inv_freq(8, 100.0, factor=4.0, low_turns=10.0, high_turns=60.0, trained_positions=1000)
    assert torch.allclose(g[0], f[0]) and torch.allclose(g[3], f[3] / 4)
    keep = (1000 * 0.1 / (2 * 3.141592653589793) - 10) / 50
    assert abs(float(g[2]) - (0.1 * keep + 0.025 * (1 - keep))) < 1e-8
    assert paged.rope_inv_freq(0).shape == (0,)
    for bad in (dict(rotary_dim=7), dict(rotary_dim=8, theta=0.0), dict(rotary_dim=8, factor=0.0),
                dict(rotary_dim=8, factor=2.0, low_turns=1.0), dict(rotary_dim=8, proportion=1.5)):
        with pytest.raises(ValueError):
            paged.rope_inv_freq(**bad)
