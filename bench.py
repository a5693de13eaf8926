#!/usr/bin/env python
"""Benchmark of the self-play training hot path: one training iteration per GPU, scaled out by data parallelism.

One step = one training iteration per GPU: a 128-decision rollout over 32,768 fights (policy
forward, simulator decision, resets), return normalisation, GAE and the PPO update (4 epochs x 8
minibatches of 524,288 samples). Metric: env-steps/s = fights x horizon x GPUs / iteration time
(a step of an environment is one policy decision, src/full_move_train.cpp:1499).

  python bench.py [--gpus N] [--steps K] [--warmup W] [--impl ours|reference]
Under torchrun each rank drives one GPU with its own fights (seed offset by rank) and the
gradient, KL and rollout statistics are summed over NCCL; rank 0 prints one JSON line.
"""
from __future__ import annotations

import argparse
import json
import lzma
import os
import statistics
import subprocess
import sys
import threading
import time
from pathlib import Path

ROOT = Path(__file__).resolve().parent
sys.path.insert(0, str(ROOT))
sys.path.insert(0, str(ROOT / "tekken8-agent_b200"))

METRIC = "env-steps/s (sim+PPO, whole box) at 32,768 fights/GPU, 1/2/4/8 B200"


def parse():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=3)
    ap.add_argument("--warmup", type=int, default=3)
    ap.add_argument("--impl", choices=("ours", "reference"), default="ours")
    ap.add_argument("--envs", type=int, default=32768)
    ap.add_argument("--horizon", type=int, default=128)
    ap.add_argument("--epochs", type=int, default=4)
    ap.add_argument("--minibatches", type=int, default=8)
    ap.add_argument("--no-cpu-baseline", action="store_true")
    ap.add_argument("--batch", type=int, default=32768, help="mlp workload: rows (config 3: 32,768)")
    ap.add_argument("--fights", type=int, default=1024, help="engine workload: fights (config 1: 1,024)")
    ap.add_argument("--frames", type=int, default=3600, help="engine workload: frames per fight (config 1: 3,600)")
    ap.add_argument("--comm", choices=("native", "torch"), default="native",
                    help="data-parallel exchanges: the library's NCCL communicator (native) or torch.distributed")
    ap.add_argument("--self-play", action="store_true",
                    help="mirror self-play: a frozen copy of the initial policy plays the other side")
    ap.add_argument("--workload", choices=("iteration", "mlp", "gae_loss", "engine"), default="iteration",
                    help="iteration: the self-play training iteration (config 4, the headline); mlp: policy forward "
                         "+ backward on one batch of 32,768 at the microbench shapes (config 3: 128 observations, 256 "
                         "candidates x 48 features, 2 x 512 hidden); gae_loss: GAE + advantage normalisation + the "
                         "clipped PPO objective over a T=128 x N=32,768 rollout with 256 slots (config 2); engine: "
                         "1,024 fights x 3,600 frames of random legal play (config 1)")
    return ap.parse_args()


def roster_raw():
    return lzma.decompress((ROOT / "tests" / "golden" / "roster41.bin.xz").read_bytes())


class ClockSampler:
    """nvidia-smi samples of SM clock and throttle reasons during the timed region. One process
    samples every GPU of the job (local rank 0 passes them all), so N ranks do not start N
    pollers of the driver."""

    FIELDS = ("index,clocks.sm,clocks.max.sm,power.draw,clocks_event_reasons.active,clocks_event_reasons.hw_slowdown,"
              "clocks_event_reasons.hw_thermal_slowdown,clocks_event_reasons.sw_thermal_slowdown,"
              "clocks_event_reasons.sw_power_cap")

    def __init__(self, indices):
        self.indices = list(indices)
        self.rows = []
        self.proc = None

    def __enter__(self):
        if not self.indices:
            return self
        try:
            self.proc = subprocess.Popen(["nvidia-smi", "-i", ",".join(map(str, self.indices)),
                                          f"--query-gpu={self.FIELDS}", "--format=csv,noheader,nounits", "-lms", "200"],
                                         stdout=subprocess.PIPE, stderr=subprocess.DEVNULL, text=True)
            self.thread = threading.Thread(target=self._read, daemon=True)
            self.thread.start()
        except OSError:
            self.proc = None
        return self

    def _read(self):
        for line in self.proc.stdout:
            parts = [p.strip() for p in line.split(",")]
            if len(parts) == 9:
                self.rows.append(parts)

    def __exit__(self, *exc):
        if self.proc is not None:
            self.proc.terminate()
            try:
                self.proc.wait(timeout=5)
            except subprocess.TimeoutExpired:
                self.proc.kill()

    def summary(self):
        if not self.rows:
            return {"sm_mhz": None, "sm_max_mhz": None, "reasons": ["unsampled"]}
        number = lambda v: v.replace(".", "").isdigit()
        sm = [float(r[1]) for r in self.rows if number(r[1])]
        mx = [float(r[2]) for r in self.rows if number(r[2])]
        names = ("hw_slowdown", "hw_thermal_slowdown", "sw_thermal_slowdown", "sw_power_cap")
        reasons = sorted({names[i] for r in self.rows for i in range(4) if r[5 + i].lower() == "active"})
        loaded = [s for s in sm if s > 0]
        out = {"sm_mhz": statistics.median(loaded) if loaded else None, "sm_max_mhz": max(mx) if mx else None,
               "reasons": reasons, "samples": len(self.rows)}
        if len(self.indices) > 1:
            per = {}
            for r in self.rows:
                if number(r[1]) and float(r[1]) > 0:
                    per.setdefault(r[0], []).append(float(r[1]))
            out["sm_mhz_per_gpu"] = {k: statistics.median(v) for k, v in sorted(per.items())}
        return out


def distributed():
    world = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    local = int(os.environ.get("LOCAL_RANK", "0"))
    return world, rank, local


def measured_peaks():
    path = ROOT / "MEASURED_PEAKS.json"
    if path.exists():
        data = json.loads(path.read_text())
        return data.get("hbm_gbs", 6650.0), data.get("bf16_tflops", 1590.0), data.get("bf16_tflops_sustained", 1400.0), "measured"
    return 6650.0, 1590.0, 1400.0, "fallback"


def max_over_ranks(values, device):
    """Each value's maximum over the ranks of the default process group (values unchanged when
    not distributed)."""
    import torch
    import torch.distributed as dist
    if not (dist.is_available() and dist.is_initialized()) or dist.get_world_size() == 1:
        return list(values)
    t = torch.tensor(values, dtype=torch.float64, device=device)
    dist.all_reduce(t, op=dist.ReduceOp.MAX)
    return t.tolist()


def reference_missing():
    """Why the reference's CPU library cannot be had (None where it can)."""
    from oracle import ref
    if ref.LIB.exists() or (ref.REFERENCE / "src").exists():
        return None
    return "the reference's CPU library is not built and its sources are not here"


def cpu_baseline(args, features, env, sample_envs=2048, sample_horizon=16):
    """The CPU leg on the host cores, on a bounded sample of the same workload."""
    missing = reference_missing()
    if missing:
        return {"unavailable": missing}
    from oracle.cpu_iteration import CpuIteration
    threads = os.cpu_count() or 1
    it = CpuIteration(roster_raw(), features, env, sample_envs, sample_horizon, args.epochs, args.minibatches,
                      threads=threads)
    seconds = it.iterate()
    value = sample_envs * sample_horizon / seconds
    return {"value": value, "unit": "env-steps/s", "cores": threads, "kind": "port",
            "sample": f"{sample_envs} fights x {sample_horizon} decisions, one iteration: the reference's CPU "
                      f"environment contract (oracle/_ref, {threads} threads) + a float32 numpy port of the policy, "
                      f"PPO objective, backward and Adam ({args.epochs} epochs x {args.minibatches} minibatches)"}


# Algorithmic work of the hot kernels, per unit they process, for the roofline figures.
# Frame step (k_step): the per-env-step bytes of a decision at the engine boundary: state in and
# out 2 x 280, noise levels 16, action 8, observations 2 x 151 x 4, masks 2 x 368 (uint8),
# reward and flags 14, table ids 8 = 2,550 B.
STEP_BYTES_PER_ENV = 2550
OBS, HIDDEN, OUTPUTS = 151, 512, 33
# GEMM FLOPs per sample, unpadded shapes (obs 151 -> 512 -> 512 -> 33).
GEMM_FLOPS_PER_SAMPLE = {
    "gemm_forward_hidden": 2 * (OBS * HIDDEN + HIDDEN * HIDDEN),
    "gemm_forward_output": 2 * HIDDEN * OUTPUTS,
    "gemm_weight_grad": 2 * (OBS * HIDDEN + HIDDEN * HIDDEN + HIDDEN * OUTPUTS),
    "gemm_input_grad": 2 * (HIDDEN * OUTPUTS + HIDDEN * HIDDEN),
}
# GEMM algorithmic bytes per sample (bf16 activations, weights negligible): the operand rows each
# GEMM must read and the epilogue rows it must write. At K = 512 every label has less than the
# B200's ridge intensity (about 220 FLOP/B against the measured peaks), so each is bound by HBM:
#   forward hidden: x 384 + h1 1,024 written, h1 1,024 read + h2 1,024 written = 3,456
#   forward output: h2 1,024 read + outputs 64 x 4 written = 1,280
#   weight gradients: (h2 1,024 + dO 128) + (dZ2 1,024 + h1 1,024) + (dZ1 1,024 + x 384) = 4,608
#   input gradients: (dO 128 + h2 1,024 + dZ2 1,024 written) + (dZ2 1,024 + h1 1,024 + dZ1 1,024 written) = 5,248
GEMM_BYTES_PER_SAMPLE = {"gemm_forward_hidden": 3456, "gemm_forward_output": 1280, "gemm_weight_grad": 4608,
                         "gemm_input_grad": 5248}
# The rollout's fused forward (k_forward_tc: normalise, both hidden layers and the output layer
# in one kernel, activations in shared memory): the three layers' FLOPs over the observation row
# read (151 x 4) and the output row written (64 x 4); the weights come from L2.
GEMM_FLOPS_PER_SAMPLE["k_forward_tc"] = GEMM_FLOPS_PER_SAMPLE["gemm_forward_hidden"] + GEMM_FLOPS_PER_SAMPLE["gemm_forward_output"]
GEMM_BYTES_PER_SAMPLE["k_forward_tc"] = OBS * 4 + 64 * 4
# GAE: read reward, value, next value (4 B each), terminated, truncated (1 B each); write
# advantage and return (4 B each) = 22 B per sample.
GAE_BYTES_PER_SAMPLE = 22
# Config 2 objective on raw logits (K = 256): read K + 1 outputs, K mask bytes, the action and four
# scalars (old log-prob, old value, advantage, return); write K + 1 gradients = 2,336 B per sample.
LOGIT_LOSS_BYTES_PER_SAMPLE = 257 * 4 + 256 + 8 + 4 * 4 + 257 * 4
# PPO loss with on-chip scores: read the 33 output floats, 12 mask words, action, table id, old
# log-prob, advantage, return, old value; write the 33 output gradients = 364 B per sample.
LOSS_BYTES_PER_SAMPLE = 33 * 4 + 12 * 4 + 8 + 4 + 4 * 4 + 33 * 4 + 24


# DRAM bytes per launch (dram__bytes_read.sum + dram__bytes_write.sum) from an ncu capture of
# the kernel, scaled to one launch of this workload by the fights it processes. Writes of the
# frame step stay in the 126 MB L2 within a launch, so its DRAM traffic is mostly reads.
TRAFFIC = {"k_step": 4.968e6 * 32768 / 8192}


def kernel_table(args, profile, steps, peaks):
    """Per-kernel device time over the timed steps, with roofline fractions where the
    algorithmic work of the kernel is known."""
    peak_hbm, peak_bf16 = peaks
    n, t = args.envs, args.horizon
    rollout_samples = (t + 1) * n
    update_samples = args.epochs * t * n
    # with the fused forward the layer GEMMs run in the update only
    forward_gemm_samples = update_samples + (0 if "k_forward_tc" in profile else rollout_samples)
    samples = {"gemm_forward_hidden": forward_gemm_samples, "gemm_forward_output": forward_gemm_samples,
               "gemm_weight_grad": update_samples, "gemm_input_grad": update_samples,
               "k_forward_tc": rollout_samples}
    total = sum(ms for _, ms in profile.values()) or 1.0
    rows = []
    for label, (launches, ms) in sorted(profile.items(), key=lambda kv: -kv[1][1]):
        row = {"kernel": label, "launches_per_step": launches / steps, "ms_per_step": ms / steps,
               "share": ms / total}
        if label in GEMM_FLOPS_PER_SAMPLE:
            seconds = ms / 1000.0
            tflops = GEMM_FLOPS_PER_SAMPLE[label] * samples[label] * steps / seconds / 1e12
            gbs = GEMM_BYTES_PER_SAMPLE[label] * samples[label] * steps / seconds / 1e9
            # the binding roof is the one whose time for this work is longer
            hbm_bound = GEMM_BYTES_PER_SAMPLE[label] / (peak_hbm * 1e9) > GEMM_FLOPS_PER_SAMPLE[label] / (peak_bf16 * 1e12)
            row.update(tensor_tflops=tflops, tensor_frac=tflops / peak_bf16, hbm_gbs=gbs, hbm_frac=gbs / peak_hbm)
            if hbm_bound:
                row.update(bound="hbm", achieved=gbs, peak=peak_hbm, unit="GB/s", frac=gbs / peak_hbm)
            else:
                row.update(bound="tensor", achieved=tflops, peak=peak_bf16, unit="TFLOP/s", frac=tflops / peak_bf16)
        elif label in ("k_step", "k_gae", "k_loss"):
            per = {"k_step": STEP_BYTES_PER_ENV * n, "k_gae": GAE_BYTES_PER_SAMPLE * t * n,
                   "k_loss": LOSS_BYTES_PER_SAMPLE * n * t // args.minibatches}[label]
            gbs = per * launches / (ms / 1000.0) / 1e9
            row.update(bound="hbm", achieved=gbs, peak=peak_hbm, unit="GB/s", frac=gbs / peak_hbm)
        rows.append(row)
    return rows


def run_reference(args):
    world, rank, local = distributed()
    if rank != 0:
        return
    missing = reference_missing()
    if missing:
        print(json.dumps({"impl": "reference", "unavailable": missing}), flush=True)
        return
    # the reference arm loads only the oracle's libraries (the reference's own CPU code), no product code
    from oracle import ref
    from oracle.cpu_iteration import CpuIteration
    features = ref.RefRoster(roster_raw()).feature_tables()
    env = ref.config4_env()
    threads = os.cpu_count() or 1
    sample_envs, sample_horizon = 2048, 16
    it = CpuIteration(roster_raw(), features, env, sample_envs, sample_horizon, args.epochs, args.minibatches,
                      threads=threads)
    for _ in range(max(0, min(args.warmup, 1))):
        it.iterate()
    times = [it.iterate() for _ in range(args.steps)]
    seconds = sum(times)
    value = sample_envs * sample_horizon * args.steps / seconds
    line = {"metric": METRIC, "value": value, "unit": "env-steps/s", "n_gpus": args.gpus, "steps": args.steps,
            "warmup": args.warmup, "ms_per_step": 1000 * seconds / args.steps, "higher_is_better": True,
            "scaling": "weak", "vs_baseline": None, "dtype": "f64 engine, f32 policy", "data": "synthetic",
            "impl": "reference",
            "config": {"workload": f"self-play iteration, bounded CPU sample of config 4 ({sample_envs} fights x "
                                   f"{sample_horizon} decisions per step)", "envs": sample_envs,
                       "horizon": sample_horizon, "epochs": args.epochs, "minibatches": args.minibatches},
            "cpu_baseline": {"value": value, "unit": "env-steps/s", "cores": threads, "kind": "port",
                             "sample": f"{sample_envs} fights x {sample_horizon} decisions per step; the reference's "
                                       f"CPU environment contract (oracle/_ref) + numpy port of the PPO math"},
            "e2e": {"value": value, "unit": "env-steps/s", "h2d_bytes_per_step": 0, "d2h_bytes_per_step": 0}}
    print(json.dumps(line), flush=True)


def run_ours(args):
    import numpy as np
    import torch
    world, rank, local = distributed()
    torch.cuda.set_device(local)
    comm = None
    if world > 1:
        import torch.distributed as dist
        from datetime import timedelta
        dist.init_process_group("nccl", timeout=timedelta(seconds=600), device_id=torch.device(f"cuda:{local}"))
        from t8b.policy import NativeComm, TorchComm
        # native: the library's own NCCL communicator, all-reduces queued from C on its stream;
        # torch: the same hooks through torch.distributed (a Python callback per exchange)
        comm = NativeComm() if args.comm == "native" else TorchComm()
    from t8b import roster as roster_module
    from t8b.train import SelfPlayTrainer
    from t8b.sim import GpuFullMoveSimulator  # noqa: F401  (loads the library)
    from t8b import profile
    roster = roster_module.parse(roster_raw())
    opponent = None
    if args.self_play:
        import tempfile
        from t8b.policy import GpuActorCritic, actor_config
        frozen = GpuActorCritic(args.envs, actor_config(), 3)
        opponent = Path(tempfile.mkdtemp()) / f"opponent_rank{rank}.t8ppo"
        frozen.save_checkpoint(opponent)
    trainer = SelfPlayTrainer(roster, environments=args.envs, horizon=args.horizon, epochs=args.epochs,
                              minibatches=args.minibatches, seed=3, comm=comm, rank=rank, opponent=opponent)
    for _ in range(args.warmup):
        trainer.host_boundary()
        trainer.iterate()
    torch.cuda.synchronize()
    if world > 1:
        torch.distributed.barrier()
    torch.cuda.synchronize()
    device_ms = []
    rollout_ms = []
    host_queue_ms = []
    bytes_up = bytes_down = 0
    frames_before = trainer.sim.frames_simulated()
    launches_before = profile.launch_count()
    # inside the timed iterations only the dominant kernel is bracketed with events (its live
    # duration gives the roofline); events around every launch cost about 2 % of the iteration
    profile.enable(True)
    profile.only("k_step")
    # local rank 0 samples every GPU of this node's ranks (device i for local rank i, named as
    # nvidia-smi counts them when CUDA_VISIBLE_DEVICES renumbers the devices)
    local_world = int(os.environ.get("LOCAL_WORLD_SIZE", str(world)))
    visible = os.environ.get("CUDA_VISIBLE_DEVICES", "")
    physical = [v.strip() for v in visible.split(",")] if visible and all(
        v.strip().isdigit() for v in visible.split(",")) else [str(i) for i in range(local_world)]
    with ClockSampler(physical[:local_world] if local == 0 else []) as clocks:
        wall0 = time.perf_counter()
        for _ in range(args.steps):
            up, down = trainer.host_boundary()
            bytes_up += up
            bytes_down += down
            start, mid, end = (torch.cuda.Event(enable_timing=True) for _ in range(3))
            start.record()
            trainer.rollout_event = mid
            metrics = trainer.iterate()
            host_queue_ms.append(trainer.rollout_host_ms)
            end.record()
            end.synchronize()
            device_ms.append(start.elapsed_time(end))
            rollout_ms.append(start.elapsed_time(mid))
        torch.cuda.synchronize()
        if world > 1:
            torch.distributed.barrier()
        wall = time.perf_counter() - wall0
    launches = profile.launch_count() - launches_before
    timed_kernels = profile.report()
    profile.enable(False)
    profile.only(None)
    frames = trainer.sim.frames_simulated() - frames_before
    # the per-kernel table: one more iteration, untimed, with events around every launch
    profile.enable(True)
    trainer.host_boundary()
    trainer.iterate()
    kernels = profile.report()
    profile.enable(False)
    total_device = sum(device_ms)
    per_rank = [total_device / args.steps]
    if world > 1:
        gathered = [torch.zeros(1, dtype=torch.float64, device="cuda") for _ in range(world)]
        torch.distributed.all_gather(gathered, torch.tensor([total_device / args.steps], dtype=torch.float64,
                                                             device="cuda"))
        per_rank = [g.item() for g in gathered]
    total_device, wall, rollout_total = max_over_ranks([total_device, wall, sum(rollout_ms)], "cuda")
    units = args.envs * args.horizon * world * args.steps
    value = units / (total_device / 1000.0)
    e2e = units / wall
    peak_hbm, peak_bf16, peak_bf16_sustained, peak_kind = measured_peaks()
    # Kernels run inside a seconds-long step: the sustained tensor peak applies; HBM is the copy peak.
    table = kernel_table(args, kernels, 1, (peak_hbm, peak_bf16_sustained))
    timed_table = kernel_table(args, timed_kernels, args.steps, (peak_hbm, peak_bf16_sustained))
    top = timed_table[0] if timed_table else None
    roofline = None
    if top is not None and "bound" in top:
        roofline = {"kernel": top["kernel"], "bound": top["bound"], "achieved": top["achieved"], "peak": top["peak"],
                    "unit": top["unit"], "frac": top["frac"], "peak_source": f"{peak_kind} (MEASURED_PEAKS.json)"
                    if peak_kind == "measured" else "fallback", "traffic": TRAFFIC.get(top["kernel"]),
                    "avg_launch_ms": top["ms_per_step"] / top["launches_per_step"]}
    line = {
        "metric": METRIC, "value": value, "unit": "env-steps/s", "n_gpus": world, "steps": args.steps,
        "warmup": args.warmup, "ms_per_step": total_device / args.steps, "higher_is_better": True, "scaling": "weak",
        "vs_baseline": None, "dtype": "f64 engine, bf16 tensor-core policy (fp32 accumulate, fp32 master weights)",
        "data": "synthetic (41-fighter roster tables from the reference loader; random-init policy)",
        "config": {"workload": "config 4: self-play iteration, 32,768 fights/GPU, T=128, 4 epochs x 8 minibatches, "
                               "screen view + live noise, " +
                               ("mirror self-play against a frozen policy" if args.self_play else "scripted opponents"),
                   "envs_per_gpu": args.envs, "horizon": args.horizon, "epochs": args.epochs,
                   "minibatch": args.envs * args.horizon // args.minibatches, "parallelism": f"dp{world}",
                   "l2": "inputs larger than L2 (rollout buffers > 4 GB per GPU)", "target_kl": "off (full 4 epochs)",
                   "comm": args.comm if world > 1 else None},
        "phases_ms_per_step": {"rollout": rollout_total / args.steps,
                               "gae_and_update": (total_device - rollout_total) / args.steps},
        "engine_frames_per_s": frames / (total_device / 1000.0) * world,
        "e2e": {"value": e2e, "unit": "env-steps/s", "h2d_bytes_per_step": bytes_up // args.steps,
                "d2h_bytes_per_step": bytes_down // args.steps},
        "rank_ms_per_step": per_rank,
        "host": {"cpus_usable": len(os.sched_getaffinity(0)), "rollout_queue_ms_per_step":
                 sum(host_queue_ms) / len(host_queue_ms)},
        "gpu_launches": launches,
        "gpu_launches_per_step": launches / args.steps,
        "roofline": roofline,
        "kernels": [{k: (round(v, 6) if isinstance(v, float) else v) for k, v in row.items()} for row in table[:12]],
        "kernels_source": "one untimed iteration after the timed ones, CUDA events around every launch",
        "clocks": clocks.summary(),
        "last_metrics": {k: float(v) for k, v in metrics.items()},
    }
    if rank == 0:
        if world == 1 and not args.no_cpu_baseline:
            line["cpu_baseline"] = cpu_baseline(args, roster.feature_tables(), trainer.sim.config)
        print(json.dumps(line), flush=True)
    if world > 1:
        torch.distributed.barrier()
        if hasattr(comm, "close"):
            torch.cuda.synchronize()
            comm.close()
        torch.distributed.destroy_process_group()


def run_mlp(args):
    """Policy forward + backward (one PPO minibatch update: forward, objective, backward, Adam)
    on a batch (config 3: 32,768; --batch 524288 is config 4's minibatch) at the microbench
    shapes, with the GEMMs' tensor-core roofline."""
    import numpy as np
    import torch
    from t8b import profile
    from t8b.policy import GpuActorCritic, actor_config, ppo_config
    from t8b._lib import RolloutView
    batch = args.batch
    obs_size, actions, features_size, hidden = 128, 256, 48, 512
    rng = np.random.default_rng(2)
    tables = 41
    feats = np.zeros((tables, actions, features_size), np.float32)
    feats[..., 0] = rng.integers(10, 31, (tables, actions))
    feats[..., 1] = rng.integers(-15, 11, (tables, actions))
    feats[..., 2] = rng.integers(5, 41, (tables, actions))
    feats[..., 3:12] = rng.integers(-3, 4, (tables, actions, 9))
    feats[..., 12:16] = np.eye(4, dtype=np.float32)[rng.integers(0, 4, (tables, actions))]
    feats[..., 16:] = rng.normal(size=(tables, actions, 32)).astype(np.float32)
    actor = actor_config(observation_size=obs_size, action_count=actions, action_feature_size=features_size,
                         hidden_size=hidden, orthogonal_initialization=0)
    policy = GpuActorCritic(batch, actor, seed=2)
    policy.set_action_feature_tables(feats)
    d = lambda a: torch.as_tensor(a, device="cuda")
    obs = d(rng.normal(size=(batch, obs_size)).astype(np.float32))
    masks = d((rng.random((batch, actions)) < 0.3).astype(np.uint8))
    masks[:, 0] = 1
    tab = d(rng.integers(0, tables, batch).astype(np.int32))
    out = policy.forward(obs, masks, batch, seed=1, step=0, tables=tab)
    acts = out["actions"].clone()
    lp = out["log_probabilities"].clone()
    val = out["values"].clone()
    adv = d(rng.normal(size=batch).astype(np.float32))
    ret = val + d(rng.normal(scale=0.5, size=batch).astype(np.float32))
    view = RolloutView()
    view.observations, view.action_masks, view.actions = obs.data_ptr(), masks.data_ptr(), acts.data_ptr()
    view.old_log_probabilities, view.old_values = lp.data_ptr(), val.data_ptr()
    view.advantages, view.returns, view.feature_tables = adv.data_ptr(), ret.data_ptr(), tab.data_ptr()
    view.sample_count = view.environment_count = batch
    view.horizon = 1
    cfg = ppo_config(epochs=1, minibatch_size=batch, target_kl=0.0)
    for i in range(args.warmup):
        policy.update_ppo(view, cfg, shuffle_seed=i)
    torch.cuda.synchronize()
    profile.enable(True)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for i in range(args.steps):
        policy.update_ppo(view, cfg, shuffle_seed=100 + i)
    end.record()
    end.synchronize()
    kernels = profile.report()
    profile.enable(False)
    ms = start.elapsed_time(end) / args.steps
    outputs = features_size + 1
    flops = {"gemm_forward_hidden": 2 * (obs_size * hidden + hidden * hidden),
             "gemm_forward_output": 2 * hidden * outputs,
             "gemm_weight_grad": 2 * (obs_size * hidden + hidden * hidden + hidden * outputs),
             "gemm_input_grad": 2 * (hidden * outputs + hidden * hidden)}
    gemm_flops = sum(flops.values()) * batch
    gemm_ms = sum(kernels[k][1] for k in flops if k in kernels) / args.steps
    _, peak_bf16, peak_sustained, peak_kind = measured_peaks()
    achieved = gemm_flops / (gemm_ms / 1000.0) / 1e12
    line = {"metric": f"policy fwd+bwd samples/s, batch {batch:,}, config-3 shapes", "value": batch / (ms / 1000.0),
            "unit": "samples/s", "n_gpus": 1, "steps": args.steps, "warmup": args.warmup, "ms_per_step": ms,
            "higher_is_better": True, "scaling": "weak", "vs_baseline": None,
            "dtype": "bf16 tensor-core products, fp32 accumulation and master weights", "data": "synthetic",
            "config": {"workload": "config 3 shapes: 128 observations -> 2 x 512 tanh -> 48-d query + value; "
                                   "256 candidate slots x 48 features per table, 41 tables, ~30% legal; one PPO "
                                   "minibatch update (forward, objective, backward, global-norm clip, Adam)",
                       "batch": batch},
            "roofline": {"kernel": "tcgen05 GEMMs (all labels)", "bound": "tensor", "achieved": achieved,
                         "peak": peak_bf16, "unit": "TFLOP/s", "frac": achieved / peak_bf16,
                         "peak_source": f"{peak_kind} burst bf16", "traffic": None,
                         "gemm_ms_per_step": gemm_ms, "gemm_gflop_per_step": gemm_flops / 1e9},
            "kernels": [{"kernel": k, "launches_per_step": v[0] / args.steps, "ms_per_step": v[1] / args.steps}
                        for k, v in sorted(kernels.items(), key=lambda kv: -kv[1][1])[:10]]}
    print(json.dumps(line), flush=True)


def clock_indices():
    visible = os.environ.get("CUDA_VISIBLE_DEVICES", "")
    if visible and all(v.strip().isdigit() for v in visible.split(",")):
        return [visible.split(",")[0].strip()]
    return ["0"]


def run_gae_loss(args):
    """Config 2: GAE with advantage normalisation and the clipped PPO objective (raw logits over
    K = 256 slots) over one rollout of T = 128 decisions x N = 32,768 fights (4,194,304 samples),
    seeded synthetic inputs (t8b.workloads.config2_rollout). A step is compute_gae(normalize) +
    t8b_ppo_output_gradient over the whole rollout; inputs (9.8 GB) are larger than L2."""
    import numpy as np
    import torch
    from t8b import profile
    from t8b.policy import GpuRolloutBuffer, ppo_config, ppo_output_gradient
    from t8b.workloads import config2_rollout
    t, n, k = args.horizon, args.envs, 256
    w = config2_rollout(t, n, k, seed=1)
    buf = GpuRolloutBuffer(n, t)
    fields = (("rewards", w.rewards), ("old_values", w.values), ("next_values", w.next_values),
              ("terminated", w.terminated), ("truncated", w.truncated))
    for name, src in fields:
        buf.tensor(name).copy_(src)
    adv = buf.tensor("advantages").reshape(-1)
    ret = buf.tensor("returns").reshape(-1)
    old_v = w.values.reshape(-1)
    cfg = ppo_config(entropy_coefficient=0.01)
    grads = torch.empty_like(w.outputs)
    sums = torch.zeros(8, dtype=torch.float64, device="cuda")
    from t8b._lib import call
    from t8b.device import ptr
    import ctypes as C

    def step():
        buf.compute_gae(0.99, 0.95, True)
        call("t8b_ppo_output_gradient", ptr(w.outputs), ptr(w.masks), ptr(w.actions), ptr(w.old_log_probabilities),
             ptr(old_v), ptr(adv), ptr(ret), w.samples, k, C.byref(cfg), ptr(grads), ptr(sums), None)

    for _ in range(args.warmup):
        step()
    torch.cuda.synchronize()
    launches_before = profile.launch_count()
    profile.enable(True)
    profile.only("k_logit_objective")
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    with ClockSampler(clock_indices()) as clocks:
        start.record()
        for _ in range(args.steps):
            step()
        end.record()
        end.synchronize()
    launches = profile.launch_count() - launches_before
    timed = profile.report()
    profile.enable(False)
    profile.only(None)
    ms = start.elapsed_time(end) / args.steps
    # per-kernel table from one more, untimed step with events around every launch
    profile.enable(True)
    step()
    kernels = profile.report()
    profile.enable(False)
    # end to end: this step's inputs copied from pinned host memory, the metric sums read back
    host_inputs = [(src, torch.empty(src.shape, dtype=src.dtype, pin_memory=True)) for src in
                   (w.rewards, w.values, w.next_values, w.terminated, w.truncated, w.outputs, w.masks, w.actions,
                    w.old_log_probabilities)]
    for src, pinned in host_inputs:
        pinned.copy_(src)
    dests = [buf.tensor("rewards"), buf.tensor("old_values"), buf.tensor("next_values"), buf.tensor("terminated"),
             buf.tensor("truncated"), w.outputs, w.masks, w.actions, w.old_log_probabilities]
    sums_host = torch.empty(8, dtype=torch.float64, pin_memory=True)
    bytes_up = sum(p.numel() * p.element_size() for _, p in host_inputs)
    torch.cuda.synchronize()
    wall0 = time.perf_counter()
    for _ in range(args.steps):
        for (_, pinned), dest in zip(host_inputs, dests):
            dest.copy_(pinned.view(dest.shape), non_blocking=True)
        torch.cuda.current_stream().synchronize()
        step()
        sums_host.copy_(sums, non_blocking=True)
        torch.cuda.synchronize()
    e2e_s = (time.perf_counter() - wall0) / args.steps
    samples = w.samples
    peak_hbm, _, _, peak_kind = measured_peaks()
    loss_launches, loss_ms = timed.get("k_logit_objective", (1, float("nan")))
    loss_avg_ms = loss_ms / max(loss_launches, 1)
    loss_gbs = LOGIT_LOSS_BYTES_PER_SAMPLE * samples / (loss_avg_ms / 1000.0) / 1e9
    rows = []
    for label, (count, total) in sorted(kernels.items(), key=lambda kv: -kv[1][1]):
        row = {"kernel": label, "launches_per_step": count, "ms_per_step": total}
        per = {"k_logit_objective": LOGIT_LOSS_BYTES_PER_SAMPLE, "k_gae": GAE_BYTES_PER_SAMPLE,
               "k_normalize": 8}.get(label)
        if per is not None:
            gbs = per * samples * count / (total / 1000.0) / 1e9
            row.update(bound="hbm", achieved=gbs, unit="GB/s", frac=gbs / peak_hbm)
        rows.append(row)
    cpu = cpu_gae_loss(w, adv, ret, cfg) if not args.no_cpu_baseline else None
    line = {"metric": f"GAE + clipped PPO loss samples/s (T={t} x N={n:,}, K={k}), 1 B200", "value": samples / (ms / 1000.0),
            "unit": "samples/s", "n_gpus": 1, "steps": args.steps, "warmup": args.warmup, "ms_per_step": ms,
            "higher_is_better": True, "scaling": "weak", "vs_baseline": None, "dtype": "f32 (fp64 statistics)",
            "data": "synthetic (seeded, t8b.workloads.config2_rollout)",
            "config": {"workload": "config 2: GAE + advantage normalisation + clipped PPO/value/entropy objective on "
                                   f"raw logits, T={t} x N={n:,}, K={k} slots ~30% legal, seed 1",
                       "samples": samples, "slots": k, "l2": "inputs larger than L2 (9.8 GB per step)"},
            "e2e": {"value": samples / e2e_s, "unit": "samples/s", "h2d_bytes_per_step": bytes_up,
                    "d2h_bytes_per_step": 64},
            "gpu_launches": launches, "gpu_launches_per_step": launches / args.steps,
            "roofline": {"kernel": "k_logit_objective", "bound": "hbm", "achieved": loss_gbs, "peak": peak_hbm,
                         "unit": "GB/s", "frac": loss_gbs / peak_hbm, "traffic": None,
                         "peak_source": f"{peak_kind} (MEASURED_PEAKS.json)", "avg_launch_ms": loss_avg_ms,
                         "algorithmic_bytes_per_sample": LOGIT_LOSS_BYTES_PER_SAMPLE},
            "kernels": rows, "kernels_source": "one untimed step after the timed ones, CUDA events around every launch",
            "clocks": clocks.summary()}
    if cpu is not None:
        line["cpu_baseline"] = cpu
    print(json.dumps(line), flush=True)


def cpu_gae_loss(w, adv, ret, cfg, sample_rows=262144):
    """CPU leg of config 2: the float64 numpy GAE restatement over the whole rollout and the
    float64 C restatement of the objective (oracle/objective.c, all host threads) over a bounded
    sample of its rows; the rate is samples / (GAE time per sample + objective time per sample)."""
    from oracle import objective
    from oracle import ppo_ref as R
    host = lambda x: x.cpu().numpy()
    rewards, values, term, trunc, nv = (host(x) for x in (w.rewards, w.values, w.terminated, w.truncated, w.next_values))
    t0 = time.perf_counter()
    a, _ = R.gae(rewards, values, term, trunc, nv, 0.99, 0.95)
    R.normalize_advantages(a)
    gae_s = (time.perf_counter() - t0) / w.samples
    rows = slice(0, sample_rows)
    inputs = [host(x[rows]) for x in (w.outputs, w.masks, w.actions, w.old_log_probabilities,
                                      w.values.reshape(-1), adv, ret)]
    threads = os.cpu_count() or 1
    t0 = time.perf_counter()
    objective.objective(*inputs, w.samples, cfg.clip_range, cfg.value_clip_range, cfg.value_coefficient,
                        cfg.entropy_coefficient, threads=threads)
    loss_s = (time.perf_counter() - t0) / sample_rows
    return {"value": 1.0 / (gae_s + loss_s), "unit": "samples/s", "cores": threads, "kind": "port",
            "sample": f"GAE + normalisation over all {w.samples} samples (numpy float64, one thread) and the objective "
                      f"over {sample_rows} of them (oracle/objective.c float64, {threads} threads)"}


def run_engine(args):
    """Config 1: 1,024 fights x 3,600 frames of the engine, every fighter picking a uniformly random
    legal candidate at each decision (PCG32 per fight), one FNV-1a state hash per fight-frame
    written to HBM. A step is one t8b_sim_random_play over the whole workload."""
    import numpy as np
    import torch
    from t8b import profile
    from t8b import roster as roster_module
    from t8b.sim import GpuFullMoveSimulator
    from t8b._lib import call
    from t8b.device import ptr
    fights, frames = args.fights, args.frames
    raw = roster_raw()
    roster = roster_module.parse(raw)
    rng = np.random.default_rng(0)
    p1 = rng.integers(0, len(roster), fights).astype(np.int32)
    p2 = rng.integers(0, len(roster), fights).astype(np.int32)
    x1 = np.full(fights, -0.45)
    x2 = np.full(fights, 0.45)
    sim = GpuFullMoveSimulator(roster, fights)
    dev = lambda a: torch.as_tensor(a, device="cuda")
    tp1, tp2, tx1, tx2 = dev(p1), dev(p2), dev(x1), dev(x2)
    hashes = torch.empty((fights, frames), dtype=torch.int64, device="cuda")

    def step(a=tp1, b=tp2, c=tx1, d=tx2, out=hashes):
        call("t8b_sim_random_play", sim._handle, fights, ptr(a), ptr(b), ptr(c), ptr(d), frames, 0, ptr(out), None)

    for _ in range(args.warmup):
        step()
    torch.cuda.synchronize()
    launches_before = profile.launch_count()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    with ClockSampler(clock_indices()) as clocks:
        start.record()
        for _ in range(args.steps):
            step()
        end.record()
        end.synchronize()
    launches = profile.launch_count() - launches_before
    ms = start.elapsed_time(end) / args.steps
    units = fights * frames
    # end to end: the matchups and start positions uploaded from pinned memory, the hashes read back
    pins = [torch.as_tensor(a).pin_memory() for a in (p1, p2, x1, x2)]
    hashes_host = torch.empty((fights, frames), dtype=torch.int64, pin_memory=True)
    torch.cuda.synchronize()
    wall0 = time.perf_counter()
    for _ in range(args.steps):
        ins = [p.to("cuda", non_blocking=True) for p in pins]
        step(*ins)
        hashes_host.copy_(hashes, non_blocking=True)
        torch.cuda.synchronize()
    e2e_s = (time.perf_counter() - wall0) / args.steps
    got = hashes.cpu().numpy().view(np.uint64)
    cpu = None
    if not args.no_cpu_baseline and not reference_missing():
        from oracle import ref
        threads = os.cpu_count() or 1
        t0 = time.perf_counter()
        want, _, _ = ref.RefRoster(raw).random_play(p1, p2, x1, x2, frames, 0, threads=threads)
        cpu_s = time.perf_counter() - t0
        cpu = {"value": units / cpu_s, "unit": "fight-frames/s", "cores": threads, "kind": "reference",
               "sample": f"the whole workload ({fights} fights x {frames} frames) on the reference's own CPU engine "
                         f"(full_core::step, oracle/_ref), one fight per thread over {threads} threads",
               "hashes_equal": bool(np.array_equal(got, want))}
    line = {"metric": f"engine fight-frames/s (random legal play, {fights:,} fights x {frames:,} frames), 1 B200",
            "value": units / (ms / 1000.0), "unit": "fight-frames/s", "n_gpus": 1, "steps": args.steps,
            "warmup": args.warmup, "ms_per_step": ms, "higher_is_better": True, "scaling": "weak",
            "vs_baseline": None, "dtype": "f64 engine (no FMA contraction)",
            "data": "synthetic (41-fighter roster tables from the reference loader; PCG32 seed 0 per fight)",
            "config": {"workload": f"config 1: engine parity run, {fights:,} fights x {frames:,} frames, per-frame state hash",
                       "fights": fights, "frames": frames,
                       "l2": "not flushed: 240 B of state per fight stays in registers; the 29 MB hash trace is "
                             "written once per step"},
            "e2e": {"value": units / e2e_s, "unit": "fight-frames/s", "h2d_bytes_per_step": fights * 24,
                    "d2h_bytes_per_step": fights * frames * 8},
            "gpu_launches": launches, "gpu_launches_per_step": launches / args.steps,
            "roofline": {"kernel": "k_random_play", "bound": "issue/latency (fp64 + integer branching)",
                         "achieved": None, "peak": None, "unit": None, "frac": None, "traffic": None,
                         "note": "one warp per fight (1,024 warps, about 7 per SM); the figure of merit is "
                                 "fight-frames/s against the CPU engine"},
            "clocks": clocks.summary()}
    if cpu is not None:
        line["cpu_baseline"] = cpu
    print(json.dumps(line), flush=True)


def main():
    args = parse()
    if args.impl == "reference":
        run_reference(args)
    elif args.workload == "mlp":
        run_mlp(args)
    elif args.workload == "gae_loss":
        run_gae_loss(args)
    elif args.workload == "engine":
        run_engine(args)
    else:
        run_ours(args)


if __name__ == "__main__":
    main()
