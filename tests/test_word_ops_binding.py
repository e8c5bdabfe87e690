"""The word operators' torch binding beside a kernel library of other headers, on the CPU."""
import os
import subprocess
import sys

from tests import words_common  # noqa: F401  (first: the binding)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_library_of_other_headers_is_refused(tmp_path):
    """A stand-in whose argument blocks have other sizes comes first in the symbol search of a fresh process."""
    src, lib = tmp_path / "other.c", tmp_path / "other.so"
    src.write_text("long long s2c_words_args_sizeof(int which) { return which == 1 ? 8 : 0; }\n")
    subprocess.check_call([os.environ.get("CC", "gcc"), "-shared", "-fPIC", str(src), "-o", str(lib)])
    load = "import ctypes, torch\nctypes.CDLL(%r, ctypes.RTLD_GLOBAL)\n" % str(lib)
    for first, said in (("import torch\n", "fine"), (load, "different headers")):
        code = first + ("try:\n    from scan2cap_amd import word_ops\n    print('fine')\n"
                        "except ImportError as e:\n    print(e)\n")
        out = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
        assert said in out.stdout, (out.stdout, out.stderr)
