"""Regenerates _constants.py (numeric values of format / data-type / enum constants) from the C
headers in ../include by compiling and running a tiny C program. Run after editing the headers:
    python cv-cuda_amd/gen_constants.py
"""
import os
import re
import subprocess
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
INC = os.path.join(os.path.dirname(HERE), "include")


def names(path, pattern):
    return re.findall(pattern, open(os.path.join(INC, path)).read(), flags=re.M)


def main():
    fmts = names("nvcv/ImageFormat.h", r"^#define (NVCV_IMAGE_FORMAT_\w+) ")
    dts = names("nvcv/DataType.h", r"^#define (NVCV_DATA_TYPE_\w+) ")
    enums = []
    for hdr in ("nvcv/DataLayout.h", "nvcv/ColorSpec.h", "nvcv/BorderType.h", "cvcuda/Types.h"):
        text = re.sub(r"/\*.*?\*/", "", open(os.path.join(INC, hdr)).read(), flags=re.S)
        for body in re.findall(r"typedef enum\s*\{(.*?)\}", text, flags=re.S):
            enums += re.findall(r"(?:^|,|\{)\s*(NVCV_[A-Za-z0-9_]+)", body, flags=re.M)
    enums = [e for e in dict.fromkeys(enums) if not e.endswith(("FORCE8", "FORCE32", "LIMIT32"))]
    src = ['#define CVCUDA_NO_HIP_HEADERS', '#include <stdio.h>', '#include <nvcv/Tensor.h>',
           '#include <nvcv/BorderType.h>', '#include <cvcuda/Types.h>', '#include <cvcuda/OpNormalize.h>',
           'int main(void){']
    dts += names("nvcv/DataType.h", r"^#define (NVCVX_DATA_TYPE_\w+) ")
    for n in fmts + dts:
        src.append('printf("%s = 0x%%016llx\\n", (unsigned long long)(%s));' % (n.split("_", 1)[1], n))
    for n in enums + ["CVCUDA_NORMALIZE_SCALE_IS_STDDEV"]:
        short = n[5:] if n.startswith("NVCV_") else n
        src.append('printf("%s = %%lld\\n", (long long)(%s));' % (short, n))
    src.append("return 0;}")
    with tempfile.TemporaryDirectory() as td:
        c = os.path.join(td, "k.c")
        open(c, "w").write("\n".join(src))
        exe = os.path.join(td, "k")
        subprocess.run(["gcc", "-std=c11", "-I" + INC, c, "-o", exe], check=True)
        out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    with open(os.path.join(HERE, "_constants.py"), "w") as f:
        f.write('"""Generated by gen_constants.py from include/*.h -- do not edit."""\n')
        f.write(out)


if __name__ == "__main__":
    main()
