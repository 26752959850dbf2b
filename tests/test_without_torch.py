"""Loading, running and building need no Torch; only ``compile`` and the operators on CUDA tensors do."""

from __future__ import annotations

import subprocess
import sys

from tests.conftest import ROOT

WITHOUT = "import sys; sys.modules['torch'] = None\n"  # every import of it raises ModuleNotFoundError


def python(code: str) -> str:
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    return done.stdout


def test_star_import_without_torch() -> None:
    names = python(WITHOUT + "from chroma_b200 import *\nprint(*sorted(n for n in dir() if not n.startswith('_')))").split()
    assert {"BatchDecoder", "Decoder", "Program", "compile", "compile_model"} <= set(names)


def test_star_import_leaves_torch_alone() -> None:
    assert python("from chroma_b200 import *\nimport sys; print('torch' in sys.modules)") == "False\n"


def test_operators_are_listed_and_imported_by_name() -> None:
    names = python("import chroma_b200; print(*dir(chroma_b200))").split()
    assert {"paged_append", "paged_attention", "step_pages", "compact_pages", "process_logits", "check_operators"} <= set(names)
    assert python("from chroma_b200 import paged_attention, process_logits; print(paged_attention.__name__)") == "paged_attention\n"
    python(WITHOUT + "import chroma_b200\ntry:\n    chroma_b200.paged_attention\nexcept ImportError:\n    pass\nelse:\n    raise SystemExit(1)")
