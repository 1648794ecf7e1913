"""What a programmatically launched kernel may read through the read-only path.

The streaming kernels of few_token.cu start while the kernel before them still runs: the router writes the ids and gates, an adapter's
shrink the rank rows `h`, the up-projection the hidden rows. `__ldg` asks for data that nobody writes while the kernel lives, and the
compiler may move such a load across the wait for the kernel before. So only the caller's operands may be read that way. The addresses
a load of `h` needs happen to depend on barriers today, so no run shows a wrong load; the source does."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "scattermoe_b200", "csrc")


def code(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def read_only_loads(text):
    """The pointer each `__ldg` reads, casts removed."""
    return [re.sub(r"reinterpret_cast<[^>]*>\(", "", a).strip().rstrip(")") for a in re.findall(r"__ldg\(((?:[^()]|\([^()]*\))*)\)", text)]


def test_only_the_callers_operands_are_read_only():
    """In the streaming kernels that is the adapters' matrix M."""
    text = code("few_token.cu")
    assert "griddepcontrol.wait" in text and "cudaLaunchAttributeProgrammaticStreamSerialization" in text
    loads = read_only_loads(text)
    assert loads and all(re.match(r"m\b", a) for a in loads), loads


def test_the_plan_reads_ids_like_any_other_memory():
    """The router may have written them just before: no promise to the compiler about the pointer."""
    text = code("few_token.cuh")
    plan = text[text.index("void make_plan("):]
    plan = plan[:plan.index("{")]
    assert "const int64_t* ids" in plan and "__restrict__" not in plan
