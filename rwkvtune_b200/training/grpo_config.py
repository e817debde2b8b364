"""``GRPOConfig`` (``rwkvtune/training/grpo_config.py:14-194``): every reference field with its default and
the same validation rules.  Fields the reference declares but never reads are accepted and ignored."""
from __future__ import annotations

import os
import warnings
from dataclasses import dataclass
from typing import Dict, List, Optional

UNUSED_FIELDS = ("delta", "kl_approximator", "top_entropy_quantile", "use_torch_compile", "generation_batch_mode",
                 "sync_ref_model", "ref_model_sync_steps", "ref_model_mixup_alpha", "mask_truncated_completions",
                 "gradient_checkpointing", "generation_batch_size", "layerwise_lr")


@dataclass
class GRPOConfig:
    n_layer: Optional[int] = None
    n_embd: Optional[int] = None
    vocab_size: Optional[int] = None
    head_size_a: Optional[int] = None
    dim_att_lora: Optional[int] = None
    dim_gate_lora: Optional[int] = None
    dim_mv_lora: Optional[int] = None
    dim_att: Optional[int] = None
    dim_ffn: Optional[int] = None
    ref_model_path: Optional[str] = None
    train_type: str = "normal"
    chunk_ctx: int = 512
    truncated_bptt: bool = True
    grad_cp: int = 0
    num_generations: int = 8
    num_iterations: int = 1
    max_prompt_length: int = 512
    max_completion_length: int = 256
    temperature: float = 1.0
    top_p: float = 1.0
    top_k: int = 0
    repetition_penalty: float = 1.0
    reward_weights: Optional[List[float]] = None
    scale_rewards: str = "group"
    advantage_clip: Optional[float] = None
    low_reward_threshold: Optional[float] = None
    low_reward_scale: float = 0.01
    loss_type: str = "dapo"
    epsilon: float = 0.2
    epsilon_high: Optional[float] = None
    delta: Optional[float] = None
    beta: float = 0.0
    kl_approximator: str = "schulman"
    importance_sampling_level: str = "token"
    top_entropy_quantile: float = 1.0
    prefill_chunk_size: int = 2048
    max_prefill_batch_size: int = -1
    max_decode_batch_size: int = -1
    logit_bias: Optional[Dict[int, float]] = None
    use_torch_compile: bool = False
    generation_batch_mode: str = "sequential"
    logprob_batch_size: Optional[int] = None
    sync_ref_model: bool = False
    ref_model_sync_steps: int = 512
    ref_model_mixup_alpha: float = 0.6
    lr_init: float = 1e-6
    lr_final: float = 1e-7
    weight_decay: float = 0.01
    warmup_steps: int = 50
    beta1: float = 0.9
    beta2: float = 0.99
    adam_eps: float = 1e-8
    grad_clip: float = 1.0
    accumulate_grad_batches: int = 1
    layerwise_lr: int = 1
    micro_bsz: int = 1
    num_workers: int = 0
    generation_batch_size: int = 8
    steps_per_generation: int = 1
    shuffle_buffer: bool = True
    accelerator: str = "gpu"
    devices: int = 1
    strategy: str = "auto"
    precision: str = "bf16"
    proj_dir: str = "output_grpo"
    seed: int = 42
    epoch_count: int = 1
    epoch_steps: Optional[int] = None
    save_every_n_batches: int = 0
    save_total_limit: int = 2
    save_optimizer_state: bool = True
    resume_from_checkpoint: Optional[str] = None
    log_steps: int = 10
    use_lora: bool = False
    lora_save_mode: str = "lora_only"
    report_to: Optional[str] = None
    run_name: Optional[str] = None
    profile_steps: int = 0   # > 0: record that many steps (after 3 warm-up steps) with torch.profiler and write <proj_dir>/profile_kernels.txt
    save_rollout_steps: int = 0
    save_rollout_path: Optional[str] = None
    mask_truncated_completions: bool = False
    gradient_checkpointing: bool = False
    log_entropy: bool = True
    ctx_len: int = 0
    ffn_precision: str = "bf16"   # "fp8": feed-forward products and activations of training in 8 bits
    grad_cp_bits: int = 16        # 8: inputs of recomputed blocks kept in 8 bits

    def __post_init__(self) -> None:
        from ..engine.engine import check_8bit_options

        check_8bit_options(self.ffn_precision, self.grad_cp_bits)
        if self.epsilon_high is None:
            self.epsilon_high = self.epsilon
        if self.num_generations <= 0:
            raise ValueError("num_generations must be > 0")
        if self.scale_rewards not in ("group", "batch", "none"):
            raise ValueError(f"scale_rewards must be group, batch or none, got {self.scale_rewards!r}")
        if self.loss_type not in ("dapo", "dr_grpo", "bnpo", "grpo"):
            raise ValueError(f"loss_type must be dapo, dr_grpo, bnpo or grpo, got {self.loss_type!r}")
        if self.importance_sampling_level not in ("token", "sequence"):
            raise ValueError("importance_sampling_level must be 'token' or 'sequence'")
        per_rollout = self.micro_bsz * self.num_generations
        if self.steps_per_generation <= 0:
            raise ValueError(f"steps_per_generation must be > 0, got {self.steps_per_generation}")
        if per_rollout < self.steps_per_generation:
            raise ValueError(f"micro_bsz x num_generations ({self.micro_bsz} x {self.num_generations} = {per_rollout}) "
                             f"must be >= steps_per_generation ({self.steps_per_generation})")
        generate_every = self.steps_per_generation * self.num_iterations
        if generate_every % self.accumulate_grad_batches:
            raise ValueError(f"generate_every ({generate_every}) must be divisible by accumulate_grad_batches "
                             f"({self.accumulate_grad_batches})")
        if self.accumulate_grad_batches > 16:
            raise ValueError(f"accumulate_grad_batches={self.accumulate_grad_batches} is too large (> 16)")
        if self.train_type == "infctx" and self.chunk_ctx <= 0:
            raise ValueError("chunk_ctx must be > 0 for infctx training")
        self.ctx_len = self.max_prompt_length + self.max_completion_length
        if self.save_rollout_steps > 0 and self.save_rollout_path is None:
            self.save_rollout_path = os.path.join(self.proj_dir, "rollouts")
        if self.report_to is not None and self.report_to not in ("swanlab", "wandb"):
            raise ValueError(f"report_to must be 'swanlab', 'wandb' or None, got {self.report_to!r}")
        if "offload" in self.strategy:
            warnings.warn("optimizer/parameter offload is accepted but not performed on B200")

    @property
    def generate_every(self) -> int:
        return self.steps_per_generation * self.num_iterations
