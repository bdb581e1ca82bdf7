"""GPT-2 training under the colocation protocol: the flow of the reference's train/gpt2.py:20-150 (model,
optimizer, text dataset of random token ids with labels = ids, micro-batch accumulation) on the HIP engine.

    python -m sirius_amd.train.gpt2 --batch-size 8 --seq-len 1024 --num-epoch 1

The reference script trains with SGD(0.1, momentum 0.9, weight decay 1e-4) at sequence length 256
(train/gpt2.py:31-32,44); `--optimizer adamw` is what the headline configuration uses.  The environment
contract and `--peer-script` are those of sirius_amd.train.resnet152.
"""
import argparse
import os
import sys
from typing import Optional

import torch

from .. import torch_col
from ..gpt2 import GPT2Engine
from ..torch_col import MemoryPool, dynamic_batch
from .common import PeerScript, attach_cu_partition, run_epochs, setup


def train(num_epoch: int, batch_size: int, global_batch_size: Optional[int] = None, dataset_size: int = 500,
          seq_len: int = 256, dtype=torch.bfloat16, optimizer: str = "sgd", peer: Optional[PeerScript] = None,
          num_distinct_samples: Optional[int] = 64, seed=0, max_grad_norm: Optional[float] = None, **model_config):
    stream = setup()
    torch_col.init_train_info(batch_size, batch_size, model_name='gpt2')
    train_mode = torch_col.get_colocate_train_mode()
    hook_mode = torch_col.get_colocate_ctrl_hook_mode()

    if torch_col.is_enable_shared_tensor():
        torch_col.tag_model_start()
    allocator = torch_col.pool_empty if torch_col.is_enable_shared_tensor() else None
    hp = dict(lr=0.1, momentum=0.9, weight_decay=1e-4) if optimizer == "sgd" else dict(lr=1e-3, weight_decay=0.01)
    model = GPT2Engine(seq_len=seq_len, dtype=dtype, optimizer=optimizer, stream=stream, allocator=allocator, **hp,
                       **model_config)
    model.init_normal(seed)
    model.set_grad_clip(max_grad_norm)
    print(f"Train params memory usage: {MemoryPool.get_memory_usage() * 1024:.2f}M")

    col_ctrl = torch_col.create_colocate_ctrl(train_mode, hook_mode, num_epoch, batch_size)
    col_ctrl.register_pytorch_hook([model])
    attach_cu_partition(model)
    enable_grad_accumulator = global_batch_size is not None or col_ctrl.train_mode.is_colocate()
    checkpoint_micro_batch = col_ctrl.train_mode.is_kill_batch()
    train_dataset, batch_manager = torch_col.init_dynamic_batch(
        dataset_size=dataset_size, dataset_type=dynamic_batch.DatasetType.TEXT_GEN,
        dataset_config=dynamic_batch.TextDatasetConfig(seq_len),
        batch_size=batch_size, global_batch_size=global_batch_size,
        enable_grad_accumulate=enable_grad_accumulator, checkpoint_micro_batch=checkpoint_micro_batch,
        lazy_batch_distributing=False, fake_data=True,
        batch_distribute_policy=dynamic_batch.BatchDistributePolicy.BY_PERFORMANCE,
        num_distinct_samples=num_distinct_samples, seed=seed)

    col_ctrl.train_start()
    torch_col.util.initialize_sgd_optimizer(model)
    grad_accumulator = torch_col.GradAccumulator(model) if batch_manager._checkpoint_micro_batch else None
    print(f'gpt2 after initialize, allocated {MemoryPool.get_allocated_memory()} '
          f'cached {MemoryPool.get_memory_usage()}', flush=True, file=sys.stderr)

    counter = {"n": 0}

    def iter_train_fn(batch: dynamic_batch.Batch):
        if peer is not None:
            peer.on_batch(counter["n"])
        counter["n"] += 1
        # labels are the ids themselves (the model shifts them); loss /= global_batch_size / batch_size
        # is folded into the loss kernel
        model.forward_backward(batch['input_ids'], loss_scale=batch_manager.loss_scale(batch))
        batch_manager.optimizer_step(batch, model, grad_accumulator=grad_accumulator)
        return 0.0

    return run_epochs("GPT2", model, iter_train_fn, col_ctrl, train_mode, num_epoch, batch_size, global_batch_size)


def main():
    parser = argparse.ArgumentParser('Train GPT-2')
    parser.add_argument('--batch-size', type=int, default=8)
    parser.add_argument('--global-batch-size', type=int, default=None)
    parser.add_argument('--num-epoch', type=int, default=1)
    parser.add_argument('--dataset-size', type=int, default=500)
    parser.add_argument('--seq-len', type=int, default=256)
    parser.add_argument('--optimizer', choices=['sgd', 'adamw'], default='sgd')
    parser.add_argument('--fp32', action='store_true')
    parser.add_argument('--fused-mlp', action='store_true', help="activation and its derivative in the MLP projections' launches")
    parser.add_argument('--max-grad-norm', type=float, default=None, help="clip the gradients' global norm ahead of every step")
    parser.add_argument('--peer-script', type=str, default='',
                        help="e.g. '10:l1:2,20:exit:8' = at micro-batch 10 send AdjustL1 to 2, at 20 InferExit to 8")
    args = parser.parse_args()
    peer = None
    if args.peer_script:
        at = {}
        for item in args.peer_script.split(','):
            idx, kind, bs = item.split(':')
            at[int(idx)] = (kind, int(bs))
        os.environ.setdefault("COLTRAIN_HAS_INFER_SERVER", "1")
        peer = PeerScript(at, verbose=True)
    print(f"GPT-2 training, batch-size={args.batch_size}, seq-len={args.seq_len}, num-epoch={args.num_epoch}")
    try:
        train(args.num_epoch, args.batch_size, global_batch_size=args.global_batch_size,
              dataset_size=args.dataset_size, seq_len=args.seq_len, optimizer=args.optimizer,
              dtype=torch.float32 if args.fp32 else torch.bfloat16, peer=peer, max_grad_norm=args.max_grad_norm,
              fused_mlp=args.fused_mlp)
    finally:
        if peer is not None:
            peer.stop()


if __name__ == '__main__':
    main()
