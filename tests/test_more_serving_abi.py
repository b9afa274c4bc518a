"""The C ABI of shared plans and attention, trims, verification and experts
without a GPU: the packed argument structs against the header's declarations,
and the refusals that come before any HIP call."""
import re
import subprocess

import pytest
import torch

import test_serving_abi
from neuralzip_amd import _native
from neuralzip_amd.gpu import serving
from test_serving_abi import HEADER, fields

STRUCTS = {"nz_pages_trim_args": _native.PAGES_TRIM, "nz_shared_plan_args": _native.SHARED_PLAN,
           "nz_shared_attention_args": _native.SHARED_ATTENTION, "nz_verify_args": _native.VERIFY,
           "nz_route_args": _native.ROUTE, "nz_expert_args": _native.EXPERTS}
ENTRIES = {"nz_pages_trim": "nz_pages_trim_args", "nz_shared_plan": "nz_shared_plan_args",
           "nz_shared_attention": "nz_shared_attention_args", "nz_verify_drafts": "nz_verify_args",
           "nz_route_experts": "nz_route_args", "nz_expert_mlp": "nz_expert_args"}


def codes(name):
    return "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([A-Za-z])", STRUCTS[name].format.lstrip("=")))


@pytest.mark.parametrize("name", STRUCTS)
def test_packed_arguments_match_the_header(name, tmp_path):
    sizes = [size for _, size in fields(name)]
    assert sizes == sorted(sizes, reverse=True)
    assert [8 if c in "qQ" else 4 for c in codes(name)] == sizes
    probe = tmp_path / "size.c"
    probe.write_text('#include <stdio.h>\n#include "neuralzip_hip.h"\n'
                     f'int main(void) {{ printf("%zu %zu %zu", sizeof({name}), sizeof(nz_shared_item), '
                     'sizeof(nz_shared_row)); return 0; }\n')
    subprocess.run(["gcc", "-std=c99", "-I", str(HEADER.parent), str(probe), "-o", str(tmp_path / "size")], check=True)
    sizes_of = subprocess.run([str(tmp_path / "size")], check=True, capture_output=True, text=True).stdout.split()
    assert int(sizes_of[0]) == STRUCTS[name].size == sum(sizes) and sizes_of[1:] == ["32", "32"]


def test_floats_and_constants_are_the_header_s():
    for name in ("nz_shared_attention_args", "nz_route_args"):
        at = [f for f, _ in fields(name)].index("scale")
        assert codes(name)[at] == "f" and codes(name).count("f") == 1
    text = HEADER.read_text()
    assert f"#define NZ_SHARED_COLUMNS {serving._COLUMNS}\n" in text
    for name, value in (("NZ_ROUTE_SOFTMAX", _native.ROUTE_SCORING["softmax"]),
                        ("NZ_ROUTE_SIGMOID", _native.ROUTE_SCORING["sigmoid"]),
                        ("NZ_EXPERT_SILU", _native.EXPERT_ACTIVATION["silu"]),
                        ("NZ_EXPERT_GELU", _native.EXPERT_ACTIVATION["gelu"])):
        assert f"{name} = {value}" in text
    # a shared plan's attention takes what the other's does, with the plan's arrays
    mine, other = ([f for f, _ in fields(n)] for n in ("nz_shared_attention_args", "nz_attention_args"))
    assert [f for f in mine if f not in ("rows", "order")] == [f for f in other if f != "counters"]
    assert mine[mine.index("items"):][:4] == ["items", "rows", "order", "partials"]


def packed(name, **values):
    names = [f for f, _ in fields(name)]
    assert set(values) <= set(names), set(values) - set(names)
    return STRUCTS[name].pack(*(4096 if values.get(f) is True else values.get(f, 0) for f in names))


TRIM = dict(lengths=True, keep=True, tables=True, free_pages=True, n_free=True, lengths_after=True, n_free_after=True,
            n_requests=4, max_pages=8, page_size=16, n_pages=32)
PLAN = dict(contexts=True, requests=True, groups=True, shared=True, items=True, rows=True, order=True,
            n_rows=10, n_requests=4, n_groups=2, n_items=32, heads=8, kv_heads=2, target=16)
ATTENTION = {k: v for k, v in dict(test_serving_abi.ATTENTION, rows=True, order=True).items() if k != "counters"}
VERIFY = dict(logits=True, draft_probs=True, tokens=True, starts=True, accept=True, sample=True, temperature=True,
              accepted=True, next=True, scratch=True, logits_row=100, draft_row=100, n_rows=5, n_requests=2, vocab=100)
ROUTE = dict(x=True, weight=True, ids=True, weights=True, scratch=True, x_row=64, tokens=3, hidden=64, experts=8, top_k=2)
EXPERTS = dict(x=True, ids=True, weights=True, gate_up=True, down=True, out=True, scratch=True, x_row=64, out_row=64,
               gate_expert=64 * 96, gate_row=64, down_expert=64 * 48, down_row=48, tokens=3, hidden=64, inter=48,
               experts=8, top_k=2, id_bytes=4)


@pytest.mark.parametrize("function, base, change, message", [
    ("nz_pages_trim", TRIM, dict(keep=0), b"Null"),
    ("nz_pages_trim", TRIM, dict(free_pages=0), b"Null"),
    ("nz_pages_trim", TRIM, dict(page_size=24), b"power of two"),
    ("nz_pages_trim", TRIM, dict(max_pages=0), b"max_pages"),
    ("nz_pages_trim", TRIM, dict(advance=2), b"advance"),
    ("nz_pages_trim", TRIM, dict(reserved=1), b"reserved"),
    ("nz_shared_plan", PLAN, dict(contexts=0), b"Null"),
    ("nz_shared_plan", PLAN, dict(items=0), b"Null"),
    ("nz_shared_plan", PLAN, dict(rows=0), b"Null"),
    ("nz_shared_plan", PLAN, dict(order=0), b"Null"),
    ("nz_shared_plan", PLAN, dict(groups=0), b"Null"),
    ("nz_shared_plan", PLAN, dict(shared=0), b"Null"),
    ("nz_shared_plan", PLAN, dict(heads=3), b"multiple of kv_heads"),
    ("nz_shared_plan", PLAN, dict(kv_heads=0), b"multiple of kv_heads"),
    ("nz_shared_plan", PLAN, dict(target=0), b"target"),
    ("nz_shared_plan", PLAN, dict(target=70000), b"target"),
    ("nz_shared_plan", PLAN, dict(n_rows=2049), b"at most"),
    ("nz_shared_plan", PLAN, dict(n_groups=1025), b"at most"),
    ("nz_shared_plan", PLAN, dict(n_items=15), b"room"),
    ("nz_shared_plan", PLAN, dict(n_requests=1 << 31), b"below 2^31"),
    ("nz_shared_plan", PLAN, dict(reserved=1), b"reserved"),
    ("nz_shared_attention", ATTENTION, dict(partials=0), b"Null"),
    ("nz_shared_attention", ATTENTION, dict(order=0), b"Null"),
    ("nz_shared_attention", ATTENTION, dict(rows=0), b"Null"),
    ("nz_shared_attention", ATTENTION, dict(heads=3), b"multiple of kv_heads"),
    ("nz_shared_attention", ATTENTION, dict(head_dim=8), b"head_dim"),
    ("nz_shared_attention", ATTENTION, dict(head_dim=272), b"head_dim"),
    ("nz_shared_attention", ATTENTION, dict(n_requests=0), b"pages and requests"),
    ("nz_shared_attention", ATTENTION, dict(n_items=1), b"fewer items"),
    ("nz_shared_attention", ATTENTION, dict(n_items=1 << 26), b"Too many"),
    ("nz_shared_attention", ATTENTION, dict(n_rows=2049, n_items=4096), b"Too many"),
    ("nz_shared_attention", ATTENTION, dict(key_slot=3), b"16 bytes"),
    ("nz_shared_attention", ATTENTION, dict(type=3), b"value type"),
    ("nz_shared_attention", ATTENTION, dict(reserved=1), b"reserved"),
    ("nz_verify_drafts", VERIFY, dict(logits=0), b"Null"),
    ("nz_verify_drafts", VERIFY, dict(tokens=0), b"Null"),
    ("nz_verify_drafts", VERIFY, dict(accept=0), b"Null"),
    ("nz_verify_drafts", VERIFY, dict(sample=0), b"Null"),
    ("nz_verify_drafts", VERIFY, dict(starts=0), b"Null"),
    ("nz_verify_drafts", VERIFY, dict(next=0), b"Null"),
    ("nz_verify_drafts", VERIFY, dict(scratch=0), b"Null"),
    ("nz_verify_drafts", VERIFY, dict(scratch=4104), b"boundary"),
    ("nz_verify_drafts", VERIFY, dict(vocab=0), b"tokens"),
    ("nz_verify_drafts", VERIFY, dict(vocab=(1 << 22) + 1), b"tokens"),
    ("nz_verify_drafts", VERIFY, dict(n_rows=65536), b"at most"),
    ("nz_verify_drafts", VERIFY, dict(n_requests=65536), b"at most"),
    ("nz_verify_drafts", VERIFY, dict(type=7), b"value type"),
    ("nz_route_experts", ROUTE, dict(x=0), b"Null"),
    ("nz_route_experts", ROUTE, dict(weights=0), b"Null"),
    ("nz_route_experts", ROUTE, dict(hidden=60), b"multiple of 8"),
    ("nz_route_experts", ROUTE, dict(hidden=0), b"multiple of 8"),
    ("nz_route_experts", ROUTE, dict(scratch=0), b"Null"),
    ("nz_route_experts", ROUTE, dict(scratch=4100), b"8-byte"),
    ("nz_route_experts", ROUTE, dict(tokens=65536), b"Too many"),
    ("nz_route_experts", ROUTE, dict(experts=1025), b"Too many"),
    ("nz_route_experts", ROUTE, dict(top_k=0), b"top_k"),
    ("nz_route_experts", ROUTE, dict(top_k=9), b"top_k"),
    ("nz_route_experts", ROUTE, dict(top_k=33, experts=40), b"top_k"),
    ("nz_route_experts", ROUTE, dict(weight=4100), b"16 bytes"),
    ("nz_route_experts", ROUTE, dict(type=1, weight_type=0), b"x's type"),
    ("nz_route_experts", ROUTE, dict(scoring=2), b"scoring"),
    ("nz_route_experts", ROUTE, dict(normalize=2), b"normalize"),
    ("nz_route_experts", ROUTE, dict(type=4), b"value type"),
    ("nz_route_experts", ROUTE, dict(reserved=1), b"reserved"),
    ("nz_expert_mlp", EXPERTS, dict(gate_up=0), b"Null"),
    ("nz_expert_mlp", EXPERTS, dict(scratch=0), b"Null"),
    ("nz_expert_mlp", EXPERTS, dict(hidden=60), b"hidden"),
    ("nz_expert_mlp", EXPERTS, dict(inter=0), b"inter"),
    ("nz_expert_mlp", EXPERTS, dict(inter=12), b"inter"),
    ("nz_expert_mlp", EXPERTS, dict(experts=0), b"experts"),
    ("nz_expert_mlp", EXPERTS, dict(experts=1025), b"experts"),
    ("nz_expert_mlp", EXPERTS, dict(top_k=33), b"choices"),
    ("nz_expert_mlp", EXPERTS, dict(top_k=0), b"choices"),
    ("nz_expert_mlp", EXPERTS, dict(id_bytes=2), b"4 or 8"),
    ("nz_expert_mlp", EXPERTS, dict(activation=2), b"activation"),
    ("nz_expert_mlp", EXPERTS, dict(tokens=1 << 22), b"Too many"),
    ("nz_expert_mlp", EXPERTS, dict(x_row=60), b"16 bytes"),
    ("nz_expert_mlp", EXPERTS, dict(down=4104), b"16 bytes"),
    ("nz_expert_mlp", EXPERTS, dict(type=3), b"value type"),
])
def test_wrong_arguments_are_refused_before_any_launch(function, base, change, message):
    lib = _native.lib()
    assert getattr(lib, function)(packed(ENTRIES[function], **dict(base, **change)), None) == -1
    assert message in lib.nz_last_error(), lib.nz_last_error()


def test_null_structs_and_calls_without_work():
    lib = _native.lib()
    for function in ENTRIES:
        assert getattr(lib, function)(None, None) == -1 and b"Null" in lib.nz_last_error()
    assert lib.nz_shared_attention(packed("nz_shared_attention_args", **dict(ATTENTION, n_rows=0, q=0)), None) == 0
    assert lib.nz_verify_drafts(packed("nz_verify_args", **dict(VERIFY, n_requests=0, starts=0)), None) == 0
    assert lib.nz_route_experts(packed("nz_route_args", **dict(ROUTE, tokens=0, x=0)), None) == 0
    assert lib.nz_expert_mlp(packed("nz_expert_args", **dict(EXPERTS, tokens=0, x=0)), None) == 0


def test_sizes_of_plans_and_scratch():
    lib = _native.lib()
    assert lib.nz_shared_items(1, 0, 32, 8, 64) == 64 and lib.nz_shared_items(0, 0, 32, 8, 64) == 64
    assert lib.nz_shared_items(65, 0, 32, 8, 64) == 128
    assert lib.nz_shared_items(64, 3, 32, 8, 64) == 192     # 64 rows' tiles, at most 3 + 8 of the groups, and half more
    for wrong in ((2049, 0, 8, 2, 1), (1, 1025, 8, 2, 1), (1, 0, 0, 1, 1), (1, 0, 8, 0, 1), (1, 0, 7, 2, 1),
                  (1, 0, 8, 2, 0)):
        assert lib.nz_shared_items(*wrong) == 0
    assert lib.nz_shared_partials(10, 32, 8, 128) == 10 * 8 * 32 * 130
    assert lib.nz_shared_partials(10, 40, 1, 64) == 10 * 2 * 32 * 66     # two blocks of columns
    assert lib.nz_shared_partials(10, 40, 0, 64) == 0
    assert lib.nz_verify_scratch(3, 2, 4097) >= (3 * 16 + 2 * 8) * 2
    assert lib.nz_expert_scratch(2, 64, 48, 3) >= 4 * 2 * 3 * 48


def test_python_entries_refuse_wrong_tensors():
    f = torch.zeros
    ints = f(3, dtype=torch.int32)
    book = serving.PageTables(3, 4, 16, 8, device="cpu")
    for bad in (f(3), f(2, dtype=torch.int32), f(3, dtype=torch.int64), f(6, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="keep"):
            book.trim(bad)
    with pytest.raises(ValueError, match="on the GPU"):
        book.trim(ints)
    with pytest.raises(ValueError, match="contexts"):
        serving.SharedPlan(ints, heads=4, kv_heads=2)           # not on the GPU
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        serving.SharedPlan(ints, heads=4, kv_heads=3)
    with pytest.raises(ValueError, match="logits"):
        serving.verify_drafts(f(2, 10), ints, ints, ints, ints)  # not on the GPU
    x, weight = f(3, 64), f(8, 64)
    with pytest.raises(ValueError, match="no backward"):
        serving.route_experts(x.clone().requires_grad_(), weight, 2)
    with pytest.raises(ValueError, match="x must be"):
        serving.route_experts(x, f(8, 56), 2)
    with pytest.raises(ValueError, match="x must be"):
        serving.route_experts(x.double(), weight.double(), 2)
    with pytest.raises(ValueError, match="contiguous, in x's dtype"):
        serving.route_experts(x, weight.half(), 2)
    with pytest.raises(ValueError, match="contiguous, in x's dtype"):
        serving.route_experts(x, f(64, 8).t(), 2)
    with pytest.raises(ValueError, match="scoring"):
        serving.route_experts(x, weight, 2, scoring="tanh")
    for k in (0, 9, 33):
        with pytest.raises(ValueError, match="top_k"):
            serving.route_experts(x, weight, k)
    with pytest.raises(ValueError, match="bias"):
        serving.route_experts(x, weight, 2, bias=f(7))
    with pytest.raises(ValueError, match="on the GPU"):
        serving.route_experts(x, weight, 2)
    ids, weights, gate_up, down = f(3, 2, dtype=torch.int32), f(3, 2), f(8, 96, 64), f(8, 64, 48)
    with pytest.raises(ValueError, match="no backward"):
        serving.expert_mlp(x, ids, weights, gate_up, down.clone().requires_grad_())
    with pytest.raises(ValueError, match="do not fit"):
        serving.expert_mlp(x, ids, weights, f(8, 90, 64), down)
    with pytest.raises(ValueError, match="do not fit"):
        serving.expert_mlp(x, ids, weights, gate_up, f(8, 56, 48))
    with pytest.raises(ValueError, match="dtype and device"):
        serving.expert_mlp(x, ids, weights, gate_up.half(), down)
    with pytest.raises(ValueError, match="Rows"):
        serving.expert_mlp(x, ids, weights, gate_up, f(8, 48, 64).transpose(1, 2))
    for bad in (ids[:2], ids.float(), f(2, 3, dtype=torch.int32).t()):
        with pytest.raises(ValueError, match="ids"):
            serving.expert_mlp(x, bad, weights, gate_up, down)
    for bad in (weights.half(), f(3, 3), f(2, 3).t()):
        with pytest.raises(ValueError, match="weights"):
            serving.expert_mlp(x, ids, bad, gate_up, down)
    with pytest.raises(ValueError, match="activation"):
        serving.expert_mlp(x, ids, weights, gate_up, down, activation="relu")
    with pytest.raises(ValueError, match="out"):
        serving.expert_mlp(x, ids, weights, gate_up, down, out=f(3, 60))
    with pytest.raises(ValueError, match="on the GPU"):
        serving.expert_mlp(x, ids, weights, gate_up, down)
