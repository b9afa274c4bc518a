"""The serving-step operators' C ABI without a GPU: the packed argument
structs against the header's declarations, and the refusals that come before
any HIP call."""
import re
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from neuralzip_amd import _native
from neuralzip_amd.gpu import serving

HEADER = Path(__file__).resolve().parents[1] / "include" / "neuralzip_hip.h"
STRUCTS = {"nz_pages_extend_args": _native.PAGES_EXTEND, "nz_pages_release_args": _native.PAGES_RELEASE,
           "nz_rotary_args": _native.ROTARY, "nz_attention_args": _native.ATTENTION,
           "nz_logits_args": _native.LOGITS}


def fields(name):
    """(field, bytes) of a struct of the header, in order."""
    body = re.search(rf"typedef struct {name} \{{(.*?)\}} {name};", HEADER.read_text(), re.S).group(1)
    out = []
    for declaration in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        declaration = declaration.strip()
        if not declaration:
            continue
        kind = re.match(r"(?:const )?\w+", declaration).group(0)
        size = 8 if "*" in declaration or "64" in kind else 4
        for field in declaration[len(kind):].replace("*", " ").split(","):
            out.append((field.strip(), size))
    return out


@pytest.mark.parametrize("name", STRUCTS)
def test_packed_arguments_match_the_header(name, tmp_path):
    """Field by field: 8-byte fields first, then 4-byte ones, and the C
    compiler's size."""
    sizes = [size for _, size in fields(name)]
    assert sizes == sorted(sizes, reverse=True)
    codes = STRUCTS[name].format.lstrip("=")
    expanded = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([A-Za-z])", codes))
    assert [8 if c in "qQ" else 4 for c in expanded] == sizes
    probe = tmp_path / "size.c"
    probe.write_text('#include <stdio.h>\n#include "neuralzip_hip.h"\n'
                     f'int main(void) {{ printf("%zu", sizeof({name})); return 0; }}\n')
    subprocess.run(["gcc", "-std=c99", "-I", str(HEADER.parent), str(probe), "-o", str(tmp_path / "size")], check=True)
    size = int(subprocess.run([str(tmp_path / "size")], check=True, capture_output=True, text=True).stdout)
    assert size == STRUCTS[name].size == sum(sizes)


def test_floats_sit_where_the_header_has_them():
    for name, field, code in (("nz_rotary_args", "eps", "ROTARY"), ("nz_attention_args", "scale", "ATTENTION")):
        at = [f for f, _ in fields(name)].index(field)
        expanded = "".join(c * int(n or 1) for n, c in
                           re.findall(r"(\d*)([A-Za-z])", getattr(_native, code).format.lstrip("=")))
        assert expanded[at] == "f" and expanded.count("f") == 1


def test_items_match_the_header():
    assert [f for f, _ in fields("nz_attention_item")] == list(_native.ATTENTION_ITEM.names)
    assert _native.ATTENTION_ITEM.itemsize == 32


def packed(name, **values):
    """A struct's bytes with the given fields and 0 elsewhere; pointers may be True (a dummy address)."""
    names = [f for f, _ in fields(name)]
    assert set(values) <= set(names), set(values) - set(names)
    return STRUCTS[name].pack(*(4096 if values.get(f) is True else values.get(f, 0) for f in names))


EXTEND = dict(lengths=True, new_tokens=True, tables=True, free_pages=True, n_free=True, slots=True, positions=True,
              requests=True, contexts=True, starts=True, status=True, lengths_after=True, n_free_after=True,
              n_requests=4, max_pages=8, page_size=16, n_pages=32, max_tokens=4)
RELEASE = dict(lengths=True, done=True, tables=True, free_pages=True, n_free=True, lengths_after=True,
               n_free_after=True, n_requests=4, max_pages=8, page_size=16, n_pages=32)
ROTARY = dict(q=True, k=True, v=True, out=True, key_cache=True, value_cache=True, cos=True, sin=True, positions=True,
              slots=True, q_token=128, q_head=64, k_token=128, k_head=64, v_token=128, v_head=64, out_token=128,
              out_head=64, key_page=2048, key_head=1024, key_slot=64, value_page=2048, value_head=1024, value_slot=64,
              tokens=3, heads=2, kv_heads=2, head_dim=64, rotary_dim=64, page_size=16, n_pages=4, n_positions=10)
ATTENTION = dict(q=True, key_cache=True, value_cache=True, out=True, tables=True, items=True, counters=True,
                 partials=True, q_row=128, q_head=64, out_row=128, out_head=64, key_page=2048, key_head=1024, key_slot=64,
                 value_page=2048, value_head=1024, value_slot=64, n_rows=2, n_items=4, heads=2, kv_heads=2, head_dim=64, n_requests=2,
                 max_pages=3, page_size=16, n_pages=4)
LOGITS = dict(logits=True, out=True, rows=2, vocab=100, logits_row=100, out_row=100)


@pytest.mark.parametrize("function, base, change, message", [
    ("nz_pages_extend", EXTEND, dict(lengths=0), b"Null"),
    ("nz_pages_extend", EXTEND, dict(slots=0), b"Null"),
    ("nz_pages_extend", EXTEND, dict(page_size=24), b"power of two"),
    ("nz_pages_extend", EXTEND, dict(page_size=8), b"power of two"),
    ("nz_pages_extend", EXTEND, dict(page_size=2048), b"power of two"),
    ("nz_pages_extend", EXTEND, dict(max_pages=0), b"max_pages"),
    ("nz_pages_extend", EXTEND, dict(max_pages=1 << 27), b"below 2^31"),
    ("nz_pages_extend", EXTEND, dict(max_tokens=1 << 31), b"below 2^31"),
    ("nz_pages_extend", EXTEND, dict(advance=2), b"advance"),
    ("nz_pages_release", RELEASE, dict(done=0), b"Null"),
    ("nz_pages_release", RELEASE, dict(page_size=0), b"power of two"),
    ("nz_pages_release", RELEASE, dict(reserved=1), b"reserved"),
    ("nz_rotary_store", ROTARY, dict(q=0), b"Null"),
    ("nz_rotary_store", ROTARY, dict(value_cache=0), b"Null"),
    ("nz_rotary_store", ROTARY, dict(slots=0), b"Null"),
    ("nz_rotary_store", ROTARY, dict(cos=0), b"Null"),
    ("nz_rotary_store", ROTARY, dict(type=3), b"value type"),
    ("nz_rotary_store", ROTARY, dict(type=1, weight_type=0), b"Norm weights"),
    ("nz_rotary_store", ROTARY, dict(head_dim=72), b"head_dim"),
    ("nz_rotary_store", ROTARY, dict(head_dim=272), b"head_dim"),
    ("nz_rotary_store", ROTARY, dict(rotary_dim=80), b"rotary_dim"),
    ("nz_rotary_store", ROTARY, dict(rotary_dim=40), b"rotary_dim"),
    ("nz_rotary_store", ROTARY, dict(kv_heads=0), b"heads"),
    ("nz_rotary_store", ROTARY, dict(k_head=60), b"16 bytes"),
    ("nz_rotary_store", ROTARY, dict(q=4098), b"16 bytes"),
    ("nz_rotary_store", ROTARY, dict(value_slot=4), b"16 bytes"),
    ("nz_rotary_store", ROTARY, dict(page_size=100), b"power of two"),
    ("nz_rotary_store", ROTARY, dict(tokens=1 << 30), b"Too many"),
    ("nz_attention", ATTENTION, dict(partials=0), b"Null"),
    ("nz_attention", ATTENTION, dict(counters=0), b"Null"),
    ("nz_attention", ATTENTION, dict(heads=3), b"multiple of kv_heads"),
    ("nz_attention", ATTENTION, dict(kv_heads=0), b"multiple of kv_heads"),
    ("nz_attention", ATTENTION, dict(head_dim=8), b"head_dim"),
    ("nz_attention", ATTENTION, dict(n_pages=0), b"pages and requests"),
    ("nz_attention", ATTENTION, dict(n_items=1), b"fewer items"),
    ("nz_attention", ATTENTION, dict(n_items=1 << 30, n_rows=1), b"Too many"),
    ("nz_attention", ATTENTION, dict(out_head=3), b"16 bytes"),
    ("nz_attention", ATTENTION, dict(type=9), b"value type"),
    ("nz_attention", ATTENTION, dict(reserved=1), b"reserved"),
    ("nz_adjust_logits", LOGITS, dict(out=0), b"Null"),
    ("nz_adjust_logits", LOGITS, dict(history=True), b"Null"),
    ("nz_adjust_logits", LOGITS, dict(history=True, lengths=True, history_bytes=2), b"4 or 8"),
    ("nz_adjust_logits", LOGITS, dict(bias_starts=True, n_bias=3), b"Null"),
    ("nz_adjust_logits", LOGITS, dict(rows=1 << 16), b"Too many"),
    ("nz_adjust_logits", LOGITS, dict(type=3), b"value type"),
])
def test_wrong_arguments_are_refused_before_any_launch(function, base, change, message):
    lib = _native.lib()
    assert getattr(lib, function)(packed(function + "_args" if function != "nz_rotary_store" and function !=
                                         "nz_adjust_logits" else {"nz_rotary_store": "nz_rotary_args",
                                                                  "nz_adjust_logits": "nz_logits_args"}[function],
                                         **dict(base, **change)), None) == -1
    assert message in lib.nz_last_error(), lib.nz_last_error()


def test_null_argument_structs_and_plans_are_refused():
    lib = _native.lib()
    for function in ("nz_pages_extend", "nz_pages_release", "nz_rotary_store", "nz_attention", "nz_adjust_logits"):
        assert getattr(lib, function)(None, None) == -1 and b"Null" in lib.nz_last_error()
    for wrong in ((None, None, 1, 1, 8, 4096, 4096), (4096, None, 1, 1, 8, None, 4096),
                  (4096, None, 1, 1, 8, 4096, None), (4096, None, 1, 0, 8, 4096, 4096),
                  (4096, None, 1, 1, 0, 4096, 4096), (4096, None, 1 << 31, 1, 8, 4096, 4096)):
        assert lib.nz_attention_plan(*wrong, None) == -1
    assert lib.nz_attention_partials(10, 32, 128) == 10 * 32 * 130


def test_calls_without_work_return_without_a_device():
    lib = _native.lib()
    assert lib.nz_rotary_store(packed("nz_rotary_args", **dict(ROTARY, tokens=0, q=0)), None) == 0
    assert lib.nz_attention(packed("nz_attention_args", **dict(ATTENTION, n_rows=0, q=0)), None) == 0
    assert lib.nz_adjust_logits(packed("nz_logits_args", **dict(LOGITS, rows=0)), None) == 0


def test_python_entries_refuse_wrong_tensors():
    f = torch.zeros
    with pytest.raises(ValueError, match="page_size"):
        serving.PageTables(2, 4, 24, 8, device="cpu")
    with pytest.raises(ValueError, match="requests"):
        serving.PageTables(0, 4, 16, 8, device="cpu")
    book = serving.PageTables(3, 4, 16, 8, device="cpu")
    assert book.free.tolist() == list(range(7, -1, -1)) and book.n_free.item() == 8
    for bad in (f(3), f(2, dtype=torch.int32), f(3, dtype=torch.int64), f(6, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="new_tokens"):
            book.extend(bad, 4)
    with pytest.raises(ValueError, match="max_tokens"):
        book.extend(f(3, dtype=torch.int32), -1)
    with pytest.raises(ValueError, match="other sizes"):
        book.extend(f(3, dtype=torch.int32), 4, out=serving.Step(3, 5, "cpu"))
    with pytest.raises(ValueError, match="done"):
        book.release(f(3))
    with pytest.raises(ValueError, match="on the GPU"):
        book.extend(f(3, dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="on the GPU"):
        book.release(f(3, dtype=torch.bool))
    with pytest.raises(ValueError, match="rotary_dim"):
        serving.Rotary(f(4, 12), f(4, 12))
    with pytest.raises(ValueError, match="cos and sin"):
        serving.Rotary(f(4, 8), f(5, 8))
    with pytest.raises(ValueError, match="one dtype"):
        serving.Rotary(f(4, 8), f(4, 8), q_weight=f(16), k_weight=f(16).half())
    rotary = serving.Rotary(f(4, 8), f(4, 8), q_weight=f(16))
    q, k, at = f(2, 4, 16), f(2, 2, 16), f(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="no backward"):
        rotary(q.clone().requires_grad_(), k, k, at)
    with pytest.raises(ValueError, match="k and v alike"):
        rotary(q, k, f(2, 1, 16), at)
    with pytest.raises(ValueError, match="do not fit"):
        rotary(q, f(3, 2, 16), f(3, 2, 16), at)
    with pytest.raises(ValueError, match="dtype and device"):
        rotary(q, k.half(), k.half(), at)
    with pytest.raises(ValueError, match="Norm weights"):
        rotary(f(2, 4, 32), f(2, 2, 32), f(2, 2, 32), at)
    with pytest.raises(ValueError, match="positions"):
        rotary(q, k, k, at.long())
    with pytest.raises(ValueError, match="contiguous"):
        rotary(f(2, 16, 4).transpose(1, 2), k, k, at)
    with pytest.raises(ValueError, match="go together"):
        rotary(q, k, k, at, slots=at.long())
    with pytest.raises(ValueError, match="Caches"):
        rotary(q, k, k, at, at.long(), f(4, 3, 16, 16), f(4, 3, 16, 16))
    for extra in ((), (at.long(), f(4, 2, 16, 16), f(4, 2, 16, 16))):
        with pytest.raises(ValueError, match="on the GPU"):
            rotary(q, k, k, at, *extra)
    with pytest.raises(ValueError, match="contexts"):
        serving.AttentionPlan(at, heads=4, kv_heads=2)   # not on the GPU
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        serving.AttentionPlan(at, heads=4, kv_heads=3)
    with pytest.raises(ValueError, match="logits"):
        serving.adjust_logits(f(2, 10))                  # not on the GPU
    assert np.dtype(_native.ATTENTION_ITEM).names[0] == "row"
