"""Host side of the losses of a projection onto a vocabulary: what a call refuses, with the
status and before anything runs, and the scratch that it asks for.  No GPU needed."""
import os
import subprocess
import sys

import pytest

import t0g

X, W, Y, LOSS, DX, DW = (0x10000000 * i for i in range(1, 7))
TEACHER, TOKENS = 0x70000000, 0x80000000


def ce(**kw):
    d = t0g.linear_ce_desc(X, W, Y, LOSS, 16, 1000, 64)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def distill(head=None, **kw):
    d = t0g.linear_distill_desc(X, W, TEACHER, TOKENS, LOSS, 16, 1000, 64, 8)
    for k, v in (head or {}).items():
        setattr(d.head, k, v)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def refused(d, *words):
    with pytest.raises(t0g.T0gError) as e:
        t0g.linear_loss_scratch_size(d)
    assert e.value.code == t0g.ERR_INVALID_ARG
    for w in words:
        assert w in str(e.value)


@pytest.mark.parametrize("change,word", [
    ({"transpose": t0g.TN}, "transpose"), ({"transpose": 9}, "transpose"), ({"label_type": 2}, "label_type"),
    ({"dx_dtype": 2}, "type"), ({"dw_dtype": 7}, "type"), ({"vocab": 0}, "size"), ({"hidden": 0}, "size"),
    ({"vocab": 1 << 31}, "size"), ({"rows": 1 << 31}, "size"),
    ({"logit_scale": 0.0}, "logit_scale"), ({"logit_scale": -1.0}, "logit_scale"),
    ({"logit_scale": float("nan")}, "logit_scale"), ({"logit_scale": float("inf")}, "logit_scale"),
    ({"ldx": 63}, "ldx"), ({"ldw": 63}, "ldw"), ({"lddx": 1}, "lddx"), ({"lddw": 63}, "lddw"),
    ({"x": 0}, "NULL"), ({"w": 0}, "NULL"), ({"loss": 0}, "NULL"), ({"labels": 0}, "labels"),
    ({"x": X + 1}, "aligned"), ({"w": W + 1}, "aligned"), ({"labels": Y + 4}, "aligned"), ({"loss": LOSS + 2}, "aligned"),
    ({"lse": DX + 2}, "aligned"), ({"dloss": DX + 1}, "aligned"), ({"dx": DX + 1}, "aligned"),
    ({"dw": DW + 2, "dw_dtype": t0g.F32}, "aligned"),
    ({"dx": X}, "overlaps"), ({"dx": X + 16 * 64 * 2 - 2}, "overlaps"), ({"dw": W}, "overlaps"), ({"lse": LOSS}, "overlaps"),
    ({"dx": DX, "dw": DX + 2}, "overlaps"), ({"loss": Y}, "overlaps"), ({"lse": W + 64}, "overlaps"),
])
def test_cross_entropy_refusals(change, word):
    refused(ce(**change), word)
    refused(distill(head={"labels": Y, **change}) if "labels" not in change else ce(**change), word)


def test_neighbours_do_not_overlap():
    assert t0g.linear_loss_scratch_size(ce(dx=X + 16 * 64 * 2, lse=LOSS + 64)) > 0


def test_nn_leading_dimension_is_the_vocabulary():
    refused(ce(transpose=t0g.NN, ldw=999), "ldw")
    assert t0g.linear_loss_scratch_size(ce(transpose=t0g.NN, ldw=1000)) > 0


@pytest.mark.parametrize("change,word", [
    ({"top_k": 0}, "top_k"), ({"top_k": 1025}, "top_k"), ({"ldt": 7}, "ldt"), ({"teacher_dtype": 2}, "teacher_dtype"),
    ({"token_type": 3}, "token_type"), ({"temperature": 0.0}, "temperature"), ({"temperature": -2.0}, "temperature"),
    ({"temperature": float("inf")}, "temperature"), ({"teacher": 0}, "NULL"), ({"tokens": 0}, "NULL"),
    ({"teacher": TEACHER + 2}, "aligned"), ({"tokens": TOKENS + 4}, "aligned"), ({"reserved": 1}, "reserved"),
    ({"teacher": LOSS}, "overlaps"), ({"tokens": LOSS}, "overlaps"),
])
def test_distill_refusals(change, word):
    refused(distill(**change), word)


def test_labels_are_optional_beside_a_teacher():
    assert t0g.linear_loss_scratch_size(distill()) > 0


def test_null_arguments():
    import ctypes
    n = ctypes.c_size_t()
    assert t0g._lib.t0g_linear_cross_entropy_scratch_size(None, ctypes.byref(n)) == t0g.ERR_INVALID_ARG
    assert t0g._lib.t0g_linear_distill_scratch_size(None, ctypes.byref(n)) == t0g.ERR_INVALID_ARG
    assert t0g._lib.t0g_linear_cross_entropy_scratch_size(ctypes.byref(ce()), None) == t0g.ERR_INVALID_ARG
    assert t0g._lib.t0g_linear_cross_entropy(None, ctypes.byref(ce())) == t0g.ERR_INVALID_ARG
    assert t0g._lib.t0g_linear_distill(None, ctypes.byref(distill())) == t0g.ERR_INVALID_ARG


def test_loss_form_refusal():
    with pytest.raises(t0g.T0gError) as e:
        t0g.set_loss_form(3)
    assert e.value.code == t0g.ERR_INVALID_ARG


def test_scratch_stays_below_the_logits():
    """8192 x 131072 logits take 4 GiB in f32 and their gradient 2 in bf16, 65536 rows eight times that; a
    piece of the vocabulary takes what it is given."""
    def scratch(rows, **kw):
        return t0g.linear_loss_scratch_size(t0g.linear_ce_desc(
            0x100000000, 0x200000000, 0x10000000, 0x20000000, rows, 131072, 4096, dx=0x300000000, dw=0x400000000, **kw))
    assert scratch(8192) < 2.5 * 2 ** 30
    assert scratch(65536) < 6 * 2 ** 30
    assert scratch(8192, max_piece=8192) < 0.75 * 2 ** 30


@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("want", ["", "x", "w", "xw"])
@pytest.mark.parametrize("rows,vocab,hidden", [
    (1, 140001, 16384), (5, 140000, 16385), (100, 140001, 16385), (129, 140000, 16385), (300, 1000003, 4097),
    (511, 32001, 100001), (2000, 140000, 16385), (3, 1 << 23, 1024), (1, (1 << 24) + 8, 512)])
def test_large_weights_of_unaligned_operands(rows, vocab, hidden, want, layout):
    """Weights of 2^31 values and more: what the unaligned products cannot take whole goes in pieces, of at most 2^30 values."""
    d = t0g.linear_ce_desc(1 << 40, 1 << 44, 1 << 30, 1 << 31, rows, vocab, hidden, transpose=layout,
                           dx=(1 << 46) * ("x" in want), dw=(1 << 48) * ("w" in want))
    assert 0 < t0g.linear_loss_scratch_size(d) < 4 << 30


@pytest.mark.parametrize("layout", ["NT", "NN"])
@pytest.mark.parametrize("want", ["", "x", "w", "xw"])
def test_hidden_states_past_31_bits(want, layout):
    """Taken with sizes that are multiples of 8, also where the last piece of the vocabulary is narrow; else refused by name."""
    def desc(rows, vocab, hidden, **kw):
        return t0g.linear_ce_desc(1 << 40, 1 << 44, 1 << 30, 1 << 31, rows, vocab, hidden, transpose=layout,
                                  dx=(1 << 46) * ("x" in want), dw=(1 << 48) * ("w" in want), **kw)
    for d in (desc(300000, 140000, 16384), desc(600000, 1000, 4096), desc(1 << 20, 264, 2056), desc(300000, 1024, 8192, ldx=8200),
              desc(300000, 1024, 8192, ldx=8193)):
        assert t0g.linear_loss_scratch_size(d) > 0
    refused(desc(300000, 32000, 8193), "x spans 2457900000")
    if layout == "NN" or "w" in want:
        refused(desc(300000, 32001, 8192), "x spans")


@pytest.mark.parametrize("hidden", [1 << 31, (1 << 32) - 8, (1 << 32) - 7, (1 << 32) - 1])
@pytest.mark.parametrize("rows", [16, 600])
def test_hidden_sizes_past_31_bits(rows, hidden):
    """Rounded up to whole 16-byte pieces the largest of them wrap to 0."""
    refused(ce(rows=rows, hidden=hidden), "size")
    refused(distill(head={"rows": rows, "hidden": hidden}), "size")


def test_no_exception_leaves_a_call():
    """A vocabulary in 2^28 pieces, whose list does not fit the memory that the process is given."""
    script = """
import resource, sys
sys.path.insert(0, sys.argv[1])
import t0g
d = t0g.linear_ce_desc(1 << 56, 1 << 58, 1 << 20, 1 << 50, 1, (1 << 31) - 1, 64, max_piece=8)
with open("/proc/self/statm") as f:
    size = int(f.read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (size + (256 << 20), size + (256 << 20)))
try:
    t0g.linear_loss_scratch_size(d)
except t0g.T0gError as e:
    print("code", e.code)
"""
    package = os.path.dirname(os.path.abspath(t0g.__file__))
    r = subprocess.run([sys.executable, "-c", script, package], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.split() == ["code", str(t0g.ERR_OUT_OF_MEMORY)], (r.returncode, r.stdout, r.stderr)
