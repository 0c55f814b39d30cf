"""Paged cache and sampling at the edges of what they take, as far as the host shows it."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "elfa_b200" / "csrc"


def test_tensor_memory_is_touched_behind_a_fence():
    """A thread that has waited for a product may read or write tensor memory behind tcgen05.fence::after_thread_sync only: in the softmax warps' code every wait for S
    or O is followed by the fence before the next access, in the order of the source."""
    text = (CSRC / "paged_prefill.cu").read_text()
    text = re.sub(r"//[^\n]*", "", text[text.index("reg_inc"):text.index("paged_prefill_join_kernel")])
    seen, open_wait = 0, False
    for word in re.findall(r"mbar_wait\(bar\(PB_[SO]FULL|tc_fence_after|tmem_(?:ld|st)\d+", text):
        if word.startswith("mbar"):
            seen, open_wait = seen + 1, True
        elif word == "tc_fence_after":
            open_wait = False
        else:
            assert not open_wait, f"{word} behind a wait without a fence"
    assert seen >= 4
