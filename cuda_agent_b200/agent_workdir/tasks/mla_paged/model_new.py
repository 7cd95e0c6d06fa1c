"""One serving step on a paged latent cache on the CUDA extension: rotation and write of the new rows, then attention.

Same constructor and forward signature as the eager model of this task; two extension calls, in the manner of the
reference's agent_workdir/model_new.py:12-13. The cache is updated in place and returned, q's last 64 columns are
overwritten with the rotated q_pe.
"""
import torch
import torch.nn as nn
import cuda_extension


class ModelNew(nn.Module):

    def __init__(self, heads: int, page: int) -> None:
        super().__init__()
        self.softmax_scale = 192 ** -0.5
        self.register_buffer("freq", 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32))

    def forward(self, q, q_pe, c_kv, k_pe, cache, page_table, q_start, kv_len):
        cuda_extension.mla_rope_append_forward(q_pe, c_kv, k_pe, cache, page_table, q_start, kv_len, self.freq,
                                               q[..., 512:], True)
        out, lse = cuda_extension.mla_paged_attention_forward(q, cache, page_table, q_start, kv_len, self.softmax_scale)
        return out, lse, cache
