"""What the ISA asks of a kernel's source and no run can show: checked on the text of csrc/."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stt-web_b200", "csrc")


def source(name):
    """The file without its comments."""
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", text, flags=re.S))


def test_a_warpgroup_executes_one_setmaxnreg():
    """All warps of a warpgroup must execute the same setmaxnreg: the chunk kernel's roles start at whole warpgroups, and
    each role's registers are set at one place, before its warps part."""
    text = source("kv8_prompt.cu")
    calls = re.findall(r"registers_(?:up|down)<(k\w+)>\(\)", text)
    assert sorted(calls) == ["kDequantRegs", "kMmaRegs", "kSoftmaxRegs"]
    values = dict(re.findall(r"(k\w+Warps) = (\d+)", text))
    assert int(values["kSoftmaxWarps"]) % 4 == 0 and int(values["kDequantWarps"]) % 4 == 0
    roles = re.findall(r"if \(([^{}]*)\) \{\s*registers_\w+<(\w+)>", text) + re.findall(r"(else) \{\s*registers_\w+<(\w+)>", text)
    assert sorted(roles) == [("else", "kSoftmaxRegs"), ("warp >= kMmaWarp", "kMmaRegs"),
                             ("warp >= kSoftmaxWarps && warp < kMmaWarp", "kDequantRegs")]


def test_registers_loaded_from_tensor_memory_are_tied_to_the_wait():
    """tcgen05.ld fills its registers until tcgen05.wait::ld: the compiler may move what reads them in front of a wait that
    does not name them, so every load is followed by tmem_wait_ld, the one place that waits."""
    waits = loads = 0
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith((".cu", ".cuh")):
            continue
        text = source(name)
        waits += text.count("tcgen05.wait::ld")
        for function in re.split(r"\n}\n", text):
            if "tcgen05.ld." in function:
                loads += 1
                assert "tmem_wait_ld(" in function[function.rindex("tcgen05.ld."):], name
    helper = source("tcgen05.cuh")
    bodies = re.findall(r"void tmem_wait_ld\((?:uint32_t|float) \(&r\)\[N\]\) \{(.*?)\n\}", helper, flags=re.S)
    assert len(bodies) == waits == 2 and loads >= 4
    for body in bodies:
        assert re.search(r'wait::ld.*for \(int i = 0; i < N; \+\+i\) asm volatile\("" : "\+[rf]"\(r\[i\]\)\);', body, flags=re.S)
