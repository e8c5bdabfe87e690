"""The word operators' torch binding on the CPU: beside a kernel library of other headers, and its answer to
arguments of types that it does not take."""
import os
import subprocess
import sys

import pytest
import torch

from tests import words_common  # noqa: F401  (first: the binding)
from scan2cap_amd import word_ops

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


_X, _T = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64)


@pytest.mark.parametrize("said,call", [
    ("tokens must be a tensor, not list", lambda: word_ops.token_scores(_X, [0, 1])),
    ("top_k", lambda: word_ops.token_scores(_X, _T, top_k=1.5)),
    ("temperature", lambda: word_ops.token_scores(_X, _T, temperature=None)),
    ("ignore_index", lambda: word_ops.token_scores(_X, _T, ignore_index=0.5)),
    ("mask must be a tensor, not list", lambda: word_ops.distill_loss(_X, _T[:, None], _X[:, :1], mask=[True, False])),
    ("temperature", lambda: word_ops.distill_loss(_X, _T[:, None], _X[:, :1], temperature="2")),
    ("scale", lambda: word_ops.embed_tokens(_T, _X, scale=None)),
    ("padding_idx", lambda: word_ops.embed_tokens(_T, _X, padding_idx=2 ** 70)),
])
def test_arguments_of_other_types_are_value_errors(said, call):
    with pytest.raises(ValueError, match=said):
        call()
