#!/usr/bin/env bash
# An MoE decoder with query / key norms, partial interleaved rotation stretched to a longer context, a sigmoid router
# over expert groups and the output layer fused with the loss, switching layouts while it trains.
#   NPROC=1 examples/intra_process/run_decoder_options.sh            (one GPU: no switches)
#   NPROC=2 examples/intra_process/run_decoder_options.sh --cpu --layers 2 --seq-length 64 --moe-ffn 128
set -euo pipefail
cd "$(dirname "$0")/../.."
NPROC="${NPROC:-1}"
STRATEGIES="${STRATEGIES:-$([ "$NPROC" -ge 2 ] && echo "ws2,ws2-ep2-etp1,ws2" || echo ws1)}"
python -m torch.distributed.run --nnodes=1 --nproc-per-node "$NPROC" --master-addr 127.0.0.1 \
  --master-port "${MASTER_PORT:-29500}" \
  examples/intra_process/train_elastic.py --model tiny-llama --num-experts 16 --moe-ffn 256 \
  --qk-layernorm --rotary-percent 0.5 --rotary-interleaved --rope-scaling yarn:4:256 \
  --router-score-function sigmoid --router-groups 4:2 --router-scaling 1.5 --fuse-linear-cross-entropy \
  --strategies "$STRATEGIES" --train-iters 10 --switch-every 3 --global-batch-size 8 "$@"
