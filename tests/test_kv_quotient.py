"""The quotient by which keys and values become SQ8 codes, on the host's IEEE arithmetic:
a product with the reciprocal, corrected once by its remainder (Markstein's method),
against the division itself for every pair of significands of a 16-bit type."""
import shutil
import subprocess

import pytest

SOURCE = r"""
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>
static float number(int exponent, uint32_t significand) { /* 1.significand (10 bits), fp16's; bf16's are among them */
    uint32_t u = (uint32_t)(127 + exponent) << 23 | significand << 13;
    float f;
    memcpy(&f, &u, 4);
    return f;
}
int main(void) {
    unsigned long pairs = 0, quotients = 0, codes = 0, plain = 0, large = 0;
    const int exponents[3] = {-63, 0, 127}; /* powers of two change nothing: the range's ends and its middle */
    for (int i = 0; i < 3; ++i)
        for (uint32_t a = 0; a < 1024; ++a) {
            const int e = exponents[i];
            const float top = number(e, a), scale = top * (1.0f / 127.0f), inverse = 1.0f / scale;
            for (int d = 0; d < 12; ++d)
                for (uint32_t b = 0; b < 1024; ++b) {
                    const float x = number(e - d, b);
                    if (x > top) continue;
                    const float want = x / scale, first = x * inverse;
                    const float q = fmaf(fmaf(-first, scale, x), inverse, first);
                    ++pairs;
                    quotients += q != want;
                    plain += first != want;
                    codes += (int)(q + 0.49999997f) != (int)roundf(want);
                    large += (int)(q + 0.49999997f) > 127;
                }
        }
    printf("%lu %lu %lu %lu %lu\n", pairs, quotients, codes, plain, large);
    return 0;
}
"""


def test_corrected_reciprocal_is_the_quotient(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    src, exe = tmp_path / "quotient.c", tmp_path / "quotient"
    src.write_text(SOURCE)
    subprocess.run(["gcc", "-O2", "-std=c11", "-ffp-contract=off", "-o", str(exe), str(src), "-lm"], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True, timeout=300).stdout
    pairs, quotients, codes, plain, large = map(int, out.split())
    assert pairs == 3 * 12059136
    assert quotients == codes == large == 0
    assert plain > 0  # the correction is needed
