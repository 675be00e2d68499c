"""CPU oracle for the b200k kernels — TEST INFRASTRUCTURE, not a product path.

Each function restates, in plain torch-on-CPU / numpy arithmetic, what the reference's
own samples and tests use as ground truth for the dense-contraction path, citing the
reference file:line it follows.  Only tests/, __graft_entry__.smoke() and bench.py's
cpu_baseline / reference arm may import this package; nothing under the b200k package
does, and the b200k operators raise when their CUDA library is missing instead of
falling back to anything here.

Pinning: oracle/quantize.py and oracle/moe.py are checked bit-for-bit against outputs of
the reference's own functions (tests/golden/*.npz, generated by tests/golden/make_golden.py
from the reference checkout) and against the reference's known-answer docstring cases;
the NVFP4 quantiser and oracle/rope.py have no counterpart in the reference and are "parity
unpinned".
"""
from .formats import *  # noqa: F401,F403
from .quantize import *  # noqa: F401,F403
from .matmul import *  # noqa: F401,F403
from .moe import *  # noqa: F401,F403
from .attention import *  # noqa: F401,F403
from .rope import *  # noqa: F401,F403
