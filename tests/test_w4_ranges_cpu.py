"""What the headers promise of the 4-bit weight calls, checked without a GPU."""
import os
import re
import subprocess

from hyacinth_b200 import api

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_type_of_bfloat16_is_a_value_of_the_enumeration(tmp_path):
    """An enumeration without a fixed type holds the values of the smallest bit field for its enumerators (up to 11: 0 .. 15); the
    conversion of any other number is undefined, and an error where a constant is wanted."""
    text = open(os.path.join(ROOT, "include", "hyacin_b200.h")).read()
    value = int(re.search(r"#define HYACIN_B200_BF16 \(\(hyacinPrecision_t\)(\d+)\)", text).group(1))
    assert value == api.BF16 and 11 < value < 16 and value % 2 == 0          # odd values are complex
    source = tmp_path / "type.cpp"
    source.write_text("#include <hyacin_b200.h>\n"
                      "constexpr int size(hyacinPrecision_t t) { switch (t) { case HYACIN_B200_BF16: return 2; default: return 0; } }\n"
                      "static_assert(size(HYACIN_B200_BF16) == 2 && size(HYACIN_F16) == 0, \"\");\n")
    subprocess.check_call(["g++", "-std=c++17", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), "-I", "/usr/local/cuda/include",
                           "-DHYACIN_BUILD_NO_NCCL", str(source)])
