"""A load from tensor memory fills its registers some time after it was issued, and the compiler does not know when: it
takes them for ready at once.  So each wait must name the registers that it makes ready; arithmetic on them could be moved in front
of one that does not."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "turbo_lossless_b200", "csrc")


def functions(text):
    """(name, arguments, body) of the device functions that hold a wait for loads from tensor memory."""
    for m in re.finditer(r"__forceinline__ void (\w+)\(([^{;]*)\)\s*\{(.*?)\n?\}\n", text, re.S):
        if "tcgen05.wait::ld" in m.group(3):
            yield m.groups()


@pytest.mark.parametrize("name", sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh"))))
def test_a_wait_names_the_registers_that_it_makes_ready(name):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    waits = list(functions(text))
    assert len(waits) == text.count("tcgen05.wait::ld.sync")          # every wait is in a function of its own
    for fn, args, body in waits:
        register = re.fullmatch(r"(?:float|uint32_t) \(&(\w+)\)\[32\]", args)
        assert register, f"{fn}({args}) does not take the registers"
        r = register.group(1)
        named = set(re.findall(r'"\+[fr]"\(' + r + r"\[(\d+)\]\)", body))
        assert named == {str(i) for i in range(32)}, f"{fn} does not name all of its registers"
