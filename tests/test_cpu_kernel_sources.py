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
