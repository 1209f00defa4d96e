"""What autograd is told of the attention operators: which arguments they change, and that they have no derivatives."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import flashoverlap_b200  # noqa: F401

OPS = torch.ops.flashoverlap_op


@pytest.mark.parametrize("name,changed", [
    ("prompt_attention", {"out"}), ("paged_attention", {"out"}), ("cache_append", {"cache"}), ("copy_pages", {"cache"}),
    ("prompt_attention_new", set()), ("paged_attention_new", set())])
def test_schemas_say_what_is_changed(name, changed):
    schema = getattr(OPS, name).default._schema
    assert schema.is_mutable == bool(changed)
    assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == changed


def test_schemas_are_what_the_wrappers_pass():
    names = [a.name for a in OPS.prompt_attention.default._schema.arguments]
    assert names == ["q", "k", "v", "out", "window", "sinks", "lengths", "scale"]
    names = [a.name for a in OPS.paged_attention.default._schema.arguments]
    assert names == ["q", "cache", "page_table", "lengths", "out", "window", "sinks", "scale"]
    names = [a.name for a in OPS.cache_append.default._schema.arguments]
    assert names == ["k", "v", "cache", "page_table", "starts", "counts"]


def test_copying_a_tensor_with_a_tangent_is_refused():
    # (the only one of the four that looks at a CPU tensor's gradients before its device)
    cache = torch.zeros(4, 8)
    with fwAD.dual_level():
        dual = fwAD.make_dual(cache, torch.ones_like(cache))
        with pytest.raises(RuntimeError, match="tangent"):
            OPS.copy_pages(dual, torch.tensor([[0, 1]]))
