"""Codes of device waits that gave up: each kernel file has its own."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nemo-c_b200", "csrc")


def test_error_codes_are_apart():
    read = lambda f: open(os.path.join(CSRC, f)).read()  # noqa: E731
    plain = re.findall(r"atomic(?:Exch|CAS)\(&g_tc_error, (?:0, )?(\d+)\)", read("k_gemm_tc.cu"))
    mx = read("k_gemm_mxfp4.cu")
    base = int(re.search(r"constexpr int ERR = (\d+);", mx).group(1))
    offsets = [int(v) for v in re.findall(r"atomicExch\(p\.err, ERR \+ (\d+)\)", mx)]
    assert mx.count("p.err,") == len(offsets) == 4 and len(plain) == 9
    assert not {base + o for o in offsets} & {int(v) for v in plain} and base > 10  # (10: the grid barrier's self-test)
