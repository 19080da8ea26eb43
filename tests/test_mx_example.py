"""The microscaled example of the integration guide, as C: it compiles with nothing declared but the pointers to device
arrays, the number of rows and the stream that it is given."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GIVEN = "int64_t M, void *d_codes, uint8_t *d_scales, void *d_w1, uint8_t *d_w1s, void *d_a, uint8_t *d_as, void *d_w2, uint8_t *d_w2s, " \
        "float *d_h, float *d_att, float *d_norm_w, float *d_shift, float *d_scale, float *d_gate, void *stream"


def test_example_compiles(tmp_path):
    text = open(os.path.join(ROOT, "INTEGRATION.md")).read().split("### Microscaled operands")[1]
    code = re.search(r"```c\n(.*?)```", text, re.S).group(1)
    src = tmp_path / "example.c"
    src.write_text("#include <stdint.h>\n#include <stddef.h>\n#include <fh3/fh3.h>\n#include <fh3/fh3_hip.h>\nvoid block(%s) {\n%s}\n" % (GIVEN, code))
    r = subprocess.run([os.environ.get("CC", "gcc"), "-std=gnu99", "-Wall", "-Werror", "-fsyntax-only", "-I" + os.path.join(ROOT, "include"),
                        str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
