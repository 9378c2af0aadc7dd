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


def test_one_corrected_product_is_the_quotient_by_7_and_by_15(tmp_path):
    """What the quantiser computes for max|w| / 7 and (hi - lo) / 15: x times the rounded reciprocal and one correction step, over all 2^23
    fractions.  The exponent of x changes nothing between the ends of the range that the kernel keeps to, so one serves, and the
    two ends themselves for good measure."""
    source = tmp_path / "quotient.cpp"
    source.write_text("""
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <initializer_list>
static float number(uint32_t bits) { float f; std::memcpy(&f, &bits, 4); return f; }
int main() {
  long wrong = 0;
  for (float by : {7.f, 15.f}) {
    const float inverse = 1.f / by;
    for (uint32_t exponent : {127u, 35u, 225u})          // 1 .. 2, from 2e-28 on, up to 6e29
      for (uint32_t fraction = 0; fraction < (1u << 23); ++fraction) {
        const float x = number(exponent << 23 | fraction), q = x * inverse;
        wrong += std::fmaf(std::fmaf(-by, q, x), inverse, q) != x / by;
      }
  }
  std::printf("%ld\\n", wrong);
}
""")
    program = tmp_path / "quotient"
    flags = ["-mfma"] if "fma" in open("/proc/cpuinfo").read() else []
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-ffp-contract=off", *flags, "-o", str(program), str(source)])
    assert subprocess.check_output([str(program)]).strip() == b"0"
