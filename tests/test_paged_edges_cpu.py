"""What the paged-cache entries promise at their edges, as far as the host shows it."""
import ctypes
import os
import re

import pytest

pytest.importorskip("torch")

from test_paged_cpu import append_args, attention_args, cache, call, paged, verify_args  # noqa: E402,F401 (a fixture)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_verification_reads_no_row_of_the_draft_before_it_is_known_to_be_needed():
    """The interface lets a sequence's last row of `draft` be missing, so the kernel may load from a row of it
    only behind the look-up that says the row is looked at.  Loads out of a buffer cannot be shown on a GPU
    without faulting it, so the order is checked in the source: of the calls that load a row's vectors, the ones
    in front of the look-up are the target's alone."""
    with open(os.path.join(ROOT, "clj-xla_b200", "csrc", "k_verify.cu")) as f:
        text = f.read()
    kernel = text[text.index("verify_rows_kernel(const"):text.index("// The race's best so far")]
    known = kernel.index("if (row - first >= count - which) return;")
    early = [m.group(0) for m in re.finditer(r"[^\n]*\bfetch\(lo \+ tid\)[^\n]*", kernel[:known])]
    assert [s.strip() for s in early] == ["if (!which) fetch(lo + tid);"]
    assert "*x" not in kernel[:known] and "x[" not in kernel[:known].replace("xv[at + u * VD_THREADS]", "")
    assert kernel.index("if (which) fetch(lo + tid);") > known


def test_attention_of_no_rows_of_a_sequence_does_nothing(paged):
    """max_tokens 0 with starts: no row is computed, nothing is enqueued (a table of more than one tile, too)."""
    lib, n = paged._library(), ctypes.c_int64(-1)
    for c in (cache(paged), cache(paged, pages_per_seq=400, page_table_stride=400)):
        a = attention_args(paged, starts=0xa0000, max_tokens=0)
        assert call(lib.attend, c, a) == (0, "")
        err = ctypes.create_string_buffer(512)
        assert lib.attend_size(ctypes.addressof(c), ctypes.addressof(a), ctypes.byref(n), err, 512) == 0 and n.value == 0


@pytest.mark.parametrize("where", ["k", "v", "q", "q_out", "inv_freq", "starts", "seq_lens", "page_table"])
@pytest.mark.parametrize("dtype,step", [("bf16", 1), ("f16", 1), ("f32", 1), ("f32", 2)])
def test_append_refuses_misaligned_pointers(paged, where, dtype, step):
    """An address between elements would be a misaligned access on the device."""
    c, a = cache(paged, dtype=paged.DTYPE_ENUM[dtype]), append_args(paged)
    s = c if hasattr(c, where) else a
    setattr(s, where, (getattr(s, where) or 0xb0000) + step)
    rc, err = call(paged._library().append, c, a)
    assert rc == 3 and where in err and "aligned" in err, (rc, err)


@pytest.mark.parametrize("where", ["starts", "seq_lens", "page_table"])
def test_attention_refuses_misaligned_pointers(paged, where):
    c, a = cache(paged), attention_args(paged)
    s = c if hasattr(c, where) else a
    setattr(s, where, (getattr(s, where) or 0xb0000) + 2)
    rc, err = call(paged._library().attend, c, a)
    assert rc == 3 and where in err and "aligned" in err, (rc, err)


@pytest.mark.parametrize("where", ["tokens_in", "starts", "uniform", "race", "tokens_out", "accepted", "logprobs", "seq_lens", "new_lens"])
def test_verify_refuses_misaligned_pointers(paged, where):
    a = verify_args(paged)
    setattr(a, where, (getattr(a, where) or 0xb0000) + 2)
    rc, err = call(paged._library().verify, a)
    assert rc == 3 and where in err and "aligned" in err, (rc, err)


def test_verify_refuses_misaligned_logits_of_the_draft(paged):
    rc, err = call(paged._library().verify, verify_args(paged, draft=0x20001))
    assert rc == 3 and "aligned" in err, (rc, err)
