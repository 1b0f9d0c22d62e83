"""MI355X-native W4A16 GEMM behind the interface of kiln's `kiln-marlin-gemm`.

* `kiln_amd.marlin_gemm`  -- `marlin_w4a16_gemm` and the `pack` namespace
  (mirror of crates/kiln-marlin-gemm/src/lib.rs)
* `kiln_amd.marlin_proj`  -- `MarlinPackedProj`, `pack_from_bf16(_batch)`,
  `matmul_bf16` (mirror of crates/kiln-model/src/marlin_proj.rs)

* `kiln_amd.lora`         -- stacked LoRA adapters fused into the GEMM epilogue
  (mirror of the call sites in crates/kiln-model/src/forward.rs:2923-2946), and
  banks of adapters that rows choose from, with their gradients
* `kiln_amd.moe`          -- a mixture-of-experts MLP on packed experts

All are thin hosts over the C ABI in include/kiln_w4a16.h; torch is used for
device memory and streams only.
"""
from . import _lib  # noqa: F401
from .marlin_gemm import marlin_w4a16_gemm, pack  # noqa: F401
from . import marlin_proj  # noqa: F401
from . import lora  # noqa: F401
from . import moe  # noqa: F401
