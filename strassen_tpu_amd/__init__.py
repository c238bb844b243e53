"""gfx950 (MI355X) tile-local one-level Strassen GEMM with fused epilogues.

Drop-in for the reference's ``strassen_pallas`` GEMM path: ``strassen_matmul``
and the relayout helpers keep the reference's names, arguments and errors;
the compute is the hand-written HIP kernel in ``csrc/strassen_gemm.hip``
behind the C ABI ``include/strassen_mi355x.h``.
"""

from .layouts import (  # noqa: F401
    is_k_contiguous, k_contiguous, rope_layout_tables, rope_layout_to_heads,
    rope_scale_layout, rope_weight_layout, swiglu_weight_layout,
)
from .strassen import (  # noqa: F401
    PROFILE_INFO, TUNED_BK, TUNED_BM, TUNED_BN, VMEM_PROFILE, check_tiling,
    cubic_matmul, native_matmul, plain_weight_kernel, strassen_kernel, strassen_matmul,
    strassen_matmul_lhs_transposed,
)

from .packing import (  # noqa: F401
    ExactSchedule, PackedOperand, SplitOperand, cache_packed_weights, cubic_weight_layout, pack_activation,
    pack_operand, packed_weight_cache_info, precision_passes, strassen_weight_layout,
)
from .strassen import PlainWeightPackWarning  # noqa: F401
from .tuning import tuned_matmul  # noqa: F401
from .paged import (  # noqa: F401
    PAGED_BAD_LENGTH, PAGED_BAD_PAGE, PAGED_OK, PAGED_OUT_OF_PAGES, PAGED_OUT_OF_ROWS, PagedPlan, paged_attention,
    paged_evict, paged_key_weights, paged_plan, paged_write,
)
from .rotary import ROTARY_SCALINGS, rotary, rotary_frequencies  # noqa: F401
from .verify import verify_drafts  # noqa: F401
from .int4 import Int4Operand, int4_matmul, int4_quantize, int4_weight_layout  # noqa: F401

__version__ = "0.5.0"
