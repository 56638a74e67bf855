"""The status word that makes the kernels' waits give up holds expired waits alone.  Whatever else a kernel notes (a page that is none, a full
table, too many landmarks) goes to a word of its own: one standing condition would otherwise cut short every long wait of every later
kernel on the device.  Read off the sources: a wait that is cut short shows itself only now and then, as a wrong result."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "landmark_attention_b200", "csrc")


def sources():
    for f in sorted(os.listdir(CSRC)):
        if f.endswith((".cu", ".cuh", ".h")):
            with open(os.path.join(CSRC, f)) as h:
                yield f, re.sub(r"//[^\n]*", "", h.read())


def test_only_expired_waits_reach_the_word_that_waits_look_at():
    seen = {}
    for f, text in sources():
        for target, code in re.findall(r"atomic(?:CAS|Exch|Or|Max)\(([^,]*status[^,]*),\s*(?:0,\s*)?(\w+)\)", text):
            seen.setdefault((target.strip(), code), []).append(f)
    # the wait itself; the two kernels that find their shared memory misplaced and return; the conditions' own word
    assert set(seen) == {("status", "where"), ("status", "kErrFwdProducer"), ("status", "kErrDqProducer"), ("status + 1", "what")}, seen


def test_conditions_are_noted():
    text = "".join(t for _, t in sources())
    codes = set(re.findall(r"note_condition\([\w.]+,\s*(\w+)\)", text))
    assert codes == {"kErrMaskGroups", "kErrSoftmaxGroups", "kBadPage", "kFull"}


def test_the_wait_looks_at_the_first_word():
    (text,) = [t for f, t in sources() if f == "sm100_ptx.cuh"]
    wait = text[text.index("void mbar_wait"):]
    wait = wait[:wait.index("\n}\n")]
    assert re.findall(r"volatile int\*>\(([^)]*)\)", wait) == ["status"]
