"""B200 (sm_100a) sparse-decode hot path of attention-lab behind a C ABI, with the reference's operator names.

`attention_lab_b200.ops` holds the drop-in operators; `attention_lab_b200.selection` the host-side plan rules;
`attention_lab_b200.install` rebinds the reference's Qwen3 wrapper to them; `attention_lab_b200.context_split` splits
one sequence's step over the ranks of a process group; `attention_lab_b200.q8` is the 8-bit K/V cache (rotary positions,
quantising write, read-back, attention with a sliding window and sinks). The C ABI is declared in `include/attention_lab_b200.h` and
built by `python -m attention_lab_b200.build`.
"""
__version__ = "0.1.0"

from .ops import (append_kvz, candidate_scores, dense_decode_step, gathered_decode_step_kernel,  # noqa: E402,F401
                  project_keys, project_queries, select_rows_kernel, sparse_decode_step_kernel)
from .q8 import Q8Cache, append_q8, attend_q8, read_q8, rotary_embed, rotary_table  # noqa: E402,F401
