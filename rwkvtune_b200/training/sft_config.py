"""``SFTConfig`` / shared training-argument record (``rwkvtune/training/sft_config.py:60-138``).

Every field of the reference is accepted with the same default.  ``strategy`` strings select the
native engines: ``auto``/``ddp`` replicate optimiser state, ``deepspeed_stage_2`` shards optimiser
state and gradients, ``deepspeed_stage_3`` also shards parameters; ``*_offload`` variants run
without offload (180 GB of HBM per GPU makes CPU offload a slowdown, not a necessity).
"""
from __future__ import annotations

import warnings
from dataclasses import dataclass
from typing import Optional

VALID_STRATEGIES = ("auto", "ddp", "deepspeed_stage_1", "deepspeed_stage_2", "deepspeed_stage_3",
                    "deepspeed_stage_2_offload", "deepspeed_stage_3_offload")


@dataclass
class SFTConfig:
    n_layer: Optional[int] = None
    n_embd: Optional[int] = None
    vocab_size: Optional[int] = None
    head_size_a: Optional[int] = None
    dim_att_lora: Optional[int] = None
    dim_gate_lora: Optional[int] = None
    dim_mv_lora: Optional[int] = None
    dim_att: Optional[int] = None
    dim_ffn: Optional[int] = None
    head_size_divisor: int = 8
    my_testing: str = "x070"
    ctx_len: int = 2048
    micro_bsz: int = 4
    num_workers: int = 0
    dataloader_shuffle: bool = True
    epoch_count: int = 10
    epoch_steps: Optional[int] = None
    epoch_save: int = 1
    save_every_n_batches: int = 0
    save_total_limit: int = 2
    save_optimizer_state: bool = True
    resume_from_checkpoint: Optional[str] = None
    accumulate_grad_batches: int = 1
    train_type: str = "normal"
    chunk_ctx: int = 512
    truncated_bptt: bool = True
    grad_cp: int = 1
    lr_init: float = 3e-4
    lr_final: float = 1e-5
    warmup_steps: int = 50
    weight_decay: float = 0.0
    layerwise_lr: int = 1
    beta1: float = 0.9
    beta2: float = 0.99
    adam_eps: float = 1e-8
    grad_clip: float = 1.0
    accelerator: str = "gpu"
    devices: int = 1
    strategy: str = "auto"
    precision: str = "bf16"
    proj_dir: str = "output_sft"
    seed: int = 42
    epoch_begin: int = 0
    use_lora: bool = False
    lora_save_mode: str = "lora_only"
    report_to: str = ""
    run_name: str = ""
    profile_steps: int = 0   # > 0: record that many steps (after 3 warm-up steps) with torch.profiler and write <proj_dir>/profile_kernels.txt
    log_every_n_steps: int = 1
    ffn_precision: str = "bf16"   # "fp8": feed-forward products and activations of training in 8 bits
    grad_cp_bits: int = 16        # 8: inputs of recomputed blocks kept in 8 bits

    def __post_init__(self) -> None:
        from ..engine.engine import check_8bit_options

        check_8bit_options(self.ffn_precision, self.grad_cp_bits)
        if self.train_type not in ("normal", "infctx"):
            raise ValueError(f"train_type must be 'normal' or 'infctx', got {self.train_type!r}")
        if self.train_type == "infctx":
            if self.chunk_ctx <= 0:
                raise ValueError("chunk_ctx must be > 0 for infctx training")
            if self.ctx_len % self.chunk_ctx:
                raise ValueError(f"ctx_len ({self.ctx_len}) must be divisible by chunk_ctx ({self.chunk_ctx})")
        if self.strategy not in VALID_STRATEGIES:
            raise ValueError(f"strategy must be one of {VALID_STRATEGIES}, got {self.strategy!r}")
        if "offload" in self.strategy:
            warnings.warn("optimizer/parameter offload is accepted but not performed on B200 (state stays in HBM)")
        if self.lora_save_mode not in ("lora_only", "full", "both"):
            raise ValueError("lora_save_mode must be lora_only, full or both")
        if self.precision not in ("fp32", "fp16", "bf16"):
            raise ValueError("precision must be fp32, fp16 or bf16")
