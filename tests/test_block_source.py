"""Rules of the block operators' kernels that no run can show without a fault:
read from the source."""
from __future__ import annotations

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "guass_b200" / "csrc"
SOURCE = (CSRC / "gfblock.cu").read_text()


def body(name: str) -> str:
    """The text of the void function ``name``, from its name to its closing brace."""
    at = re.search(r"(?:void|\)) " + name + r"\(", SOURCE).start()
    depth = 0
    for i in range(SOURCE.index("{", at), len(SOURCE)):
        depth += {"{": 1, "}": -1}.get(SOURCE[i], 0)
        if depth == 0:
            return SOURCE[at:i + 1]
    raise AssertionError(name)


def test_one_cta_group_in_a_kernel():
    """Every tcgen05 instruction of a kernel has the same cta_group, the ones behind a wait that gave up too."""
    used = re.findall(r"tc::(tmem_alloc|tmem_free|mma_commit|mma)<([^>;]*?)[,>]", body("gemm_kernel"))
    assert len(used) >= 6
    assert {group for _, group in used} == {"PAIR"}


def test_barriers_are_initialised_before_the_fence():
    text = body("gemm_kernel")
    fence = text.index("fence_barrier_init")
    inits = [m.start() for m in re.finditer("mbar_init", text)]
    assert inits and max(inits) < fence
    for bar in ("full", "empty", "acc_full", "acc_empty", "spare"):
        assert re.search(r"mbar_init\([^;]*\b" + bar + r"\b", text[:fence]), bar


def test_both_ctas_of_a_pair_stay_for_their_copies():
    """A producer that gave up outlasts its copies in flight: the first CTA waits for the stages it filled, the second,
    whose copies count on the first one's barriers, for a fixed time."""
    text = body("gemm_kernel")
    first = text.index("if (!ok && rank == 0) {")
    after = text[first:text.index("warp == 1", first)]
    assert "mbar_wait(full" in after.split("else if (!ok)")[0]
    assert "__nanosleep" in after.split("else if (!ok)")[1]


def test_the_checked_build_checks_every_source():
    from guass_b200 import _build

    for src in _build.SOURCES:
        assert _build._object(src, True) != _build._object(src, False)
        assert "GF_CHECK" in src.read_text()


def test_kernels_that_address_memory_themselves_check_their_bounds():
    for kernel in ("join_kernel", "column_sums_kernel", "column_join_kernel", "align_kernel", "skinny_kernel",
                   "dropout_kernel", "quantize_rows_kernel", "result", "fetch", "gemm_kernel"):
        assert "GFB_IN_BOUNDS" in body(kernel), kernel


def test_local_arrays_that_move_as_wide_words_are_aligned():
    """An array of 16-bit elements is 2-byte aligned by itself; a wide access to one in local memory would fault."""
    names = set(re.findall(r"reinterpret_cast<(?:const )?(?:uint|float)[24]\*>\(&?(\w+)[\[)]", SOURCE))
    local = {n for n in names if re.search(r"^\s+(?:\S+ )*T " + n + r"\[", SOURCE, flags=re.M)}
    assert {"r", "tail", "in", "add", "out", "held", "xs"} <= local
    for n in local:
        for line in re.findall(r"^.*\bT " + n + r"\[.*$", SOURCE, flags=re.M):
            assert "__align__" in line, line
