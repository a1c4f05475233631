#!/usr/bin/env python3
"""Benchmark: ProteinMPNN v_48_020 designed residues/s.

One step = one batched design over 64 synthetic backbones (generator seeds
rank*64 + 0..63) x L=256 x 32 sequences at T=0.1 with a random decoding order
per sequence: featurisation, encoder, decoder tables and the autoregressive
decode of all 2,048 sequences (524,288 designed residues per GPU).

* ``value``  -- inputs resident in HBM (hkb_mpnn_design_device); per-step
  device time from CUDA events on the launching stream (the decoding orders
  are generated on the device inside the interval); L2 flushed (512 MiB
  write) before each step.
* ``e2e``    -- the host API (hkb_mpnn_design): pinned coords/atom-sources
  uploaded and tokens + log-probs + scores read back every step; wall clock.
  The log-probs buffer is pinned, so the decode kernel writes the rows into it
  as it samples them (the same bytes cross the bus, during the kernel instead
  of in a copy after it).
* ``roofline`` -- the autoregressive decode kernel (the dominant kernel):
  algorithmic FLOPs per launch (29,103,360 per designed residue, the reference
  formulation) over its CUDA-event duration, against the measured burst 16-bit
  tensor peak of MEASURED_PEAKS.json (the kernel is timed on its own, within a
  step of a few tens of milliseconds).
* ``cpu_baseline`` -- the reference's own CPU design path (oracle/_ref, the
  reference sources compiled here) on the host cores, bounded sample.

``--impl reference`` times that reference CPU path alone on the same metric.
Where the reference's sources or the published weight image are not at hand, that
arm prints why, the sample is left out, and the engine runs on weights of random
values, as ``data`` then says.
Multi-GPU: one process per GPU (torchrun), proteins sharded by rank, no
collective on the data path (weak scaling); barrier + max-over-ranks timing.
"""
from __future__ import annotations

import argparse
import ctypes
import json
import os
import statistics
import subprocess
import sys
import threading
import time
from pathlib import Path

import numpy as np

ROOT = Path(__file__).resolve().parent
sys.path.insert(0, str(ROOT))

L_RES = 256
N_PROT = 64
N_SEQ = 32
TEMP = 0.1
FLOP_DECODE_PER_RES = 29_103_360
FLOP_ENCODE_PER_RES = 54_657_024
WEIGHTS = ROOT / "hikoboshi_b200" / "weights" / "Hikoboshi-ProteinMPNN-v48-020.safetensors"
METRIC = "ProteinMPNN v48 designed residues/sec at L=256 x32 seqs; us per decode step"


def published_weights() -> bool:
    return WEIGHTS.exists()


def engine_weights():
    """The published weight image, or one of random values where it is not at hand:
    the work does not depend on the values."""
    if published_weights():
        return WEIGHTS
    sys.path.insert(0, str(ROOT / "tests"))
    from random_weights import random_weights
    return random_weights(0)


def data_note(text: str) -> str:
    return text if published_weights() else text + "; random weights of that architecture"


def reference_missing() -> str | None:
    """Why the reference's own CPU path cannot run here, or None."""
    from oracle.oracle import REF_SO
    if not REF_SO.exists():
        return "the reference's sources are not at hand, so its CPU path is not compiled"
    return None if published_weights() else "the reference's weight image is not at hand"


def dist_env():
    return (int(os.environ.get("RANK", 0)), int(os.environ.get("WORLD_SIZE", 1)),
            int(os.environ.get("LOCAL_RANK", 0)))


def make_inputs(rank: int):
    from hikoboshi_b200 import synthetic_backbone
    cs, ss = [], []
    for i in range(N_PROT):
        c, s = synthetic_backbone(rank * N_PROT + i, L_RES)
        cs.append(c)
        ss.append(s)
    return np.concatenate(cs), np.concatenate(ss)


class ClockSampler:
    """SM clock, power and clock-event reasons sampled every 20 ms through NVML
    (nvidia_ml_py) during the timed region; nvidia-smi at 200 ms if NVML is
    not importable."""

    REASONS = {"hw_slowdown": 0x8, "hw_thermal_slowdown": 0x40,
               "sw_thermal_slowdown": 0x20, "sw_power_cap": 0x4}
    FIELDS = ("index,clocks.sm,clocks.max.sm,power.draw,clocks_event_reasons.active,"
              "clocks_event_reasons.hw_slowdown,clocks_event_reasons.hw_thermal_slowdown,"
              "clocks_event_reasons.sw_thermal_slowdown,clocks_event_reasons.sw_power_cap")

    def __init__(self, gpu_index: int):
        self.gpu = gpu_index            # CUDA ordinal; NVML is addressed by PCI bus id
        self.samples: list[tuple[float, float, int]] = []   # (sm MHz, power W, reasons)
        self.max_mhz = None
        self.proc = None
        self.stop_evt = threading.Event()
        self.thread = None
        self.backend = None

    def start(self):
        try:
            import pynvml
            pynvml.nvmlInit()
            h = None
            try:
                import torch
                pr = torch.cuda.get_device_properties(self.gpu)
                bus = f"{pr.pci_domain_id:08X}:{pr.pci_bus_id:02X}:{pr.pci_device_id:02X}.0"
                h = pynvml.nvmlDeviceGetHandleByPciBusId(bus)
            except Exception:
                h = pynvml.nvmlDeviceGetHandleByIndex(self.gpu)
            self.max_mhz = float(pynvml.nvmlDeviceGetMaxClockInfo(h, pynvml.NVML_CLOCK_SM))
            get_reasons = getattr(pynvml, "nvmlDeviceGetCurrentClocksEventReasons", None) or \
                pynvml.nvmlDeviceGetCurrentClocksThrottleReasons

            def poll():
                while not self.stop_evt.is_set():
                    try:
                        self.samples.append((
                            float(pynvml.nvmlDeviceGetClockInfo(h, pynvml.NVML_CLOCK_SM)),
                            pynvml.nvmlDeviceGetPowerUsage(h) / 1000.0, int(get_reasons(h))))
                    except Exception:
                        pass
                    self.stop_evt.wait(0.02)

            self.backend = "nvml"
            self.thread = threading.Thread(target=poll, daemon=True)
            self.thread.start()
            return
        except Exception:
            pass
        try:
            self.proc = subprocess.Popen(
                ["nvidia-smi", f"--id={self.gpu}", f"--query-gpu={self.FIELDS}",
                 "--format=csv,noheader,nounits", "-lms", "200"],
                stdout=subprocess.PIPE, stderr=subprocess.DEVNULL, text=True)
            self.backend = "nvidia-smi"
            self.thread = threading.Thread(target=self._read_smi, daemon=True)
            self.thread.start()
        except OSError:
            self.proc = None

    def _read_smi(self):
        for line in self.proc.stdout:
            f = [x.strip() for x in line.split(",")]
            if len(f) < 9:
                continue
            try:
                bits = 0
                for (n, b), v in zip(self.REASONS.items(), (f[5], f[6], f[7], f[8])):
                    if v.lower().startswith("active"):
                        bits |= b
                self.samples.append((float(f[1]), float(f[3]), bits))
                self.max_mhz = float(f[2])
            except ValueError:
                continue

    def stop(self) -> dict:
        if self.backend is None:
            return {"sm_mhz": None, "sm_max_mhz": None, "reasons": ["clock sampling unavailable"]}
        self.stop_evt.set()
        if self.proc is not None:
            self.proc.terminate()
            try:
                self.proc.wait(timeout=5)
            except subprocess.TimeoutExpired:
                self.proc.kill()
        if self.thread is not None:
            self.thread.join(timeout=5)
        sm = [x[0] for x in self.samples]
        power = [x[1] for x in self.samples]
        reasons = sorted({n for n, b in self.REASONS.items()
                          for x in self.samples if x[2] & b})
        load = [x for x, p in zip(sm, power) if p > 200] or sm
        return {"sm_mhz": statistics.median(load) if load else None, "sm_max_mhz": self.max_mhz,
                "reasons": reasons, "samples": len(sm),
                "power_w_max": max(power) if power else None, "source": self.backend}


def measured_peaks():
    p = ROOT / "MEASURED_PEAKS.json"
    if p.exists():
        d = json.loads(p.read_text())
        return d, "measured"
    return {"hbm_gbs": 6650.0, "bf16_tflops": 1590.0, "bf16_tflops_sustained": 1400.0}, "fallback"


def profiled_traffic(precision: str):
    """dram read+write bytes per launch of the decode kernel, from the
    committed ncu summary of the same workload (None if not captured)."""
    f = ROOT / "profiles" / f"ar_decode_{precision}_config2.txt"
    if not f.exists():
        return None
    for line in f.read_text().splitlines():
        if line.startswith("traffic_bytes_per_launch:"):
            return float(line.split(":", 1)[1])
    return None


def cpu_baseline_sample(threads: int, seqs_per_thread: int = 1):
    """The reference's design path (algorithms::inverse_fold_proteinmpnn_v48_020
    compiled from its sources) on `threads` host threads, each designing
    `seqs_per_thread` sequences of its own config-2 backbone (L=256, T=0.1,
    random order).  Returns (residues/s, description)."""
    from concurrent.futures import ThreadPoolExecutor
    from oracle.oracle import RefLib

    # The inputs come from the generator linked into the reference library,
    # so this leg never loads the engine library.
    ref = RefLib(WEIGHTS)
    inputs = [ref.synthetic_backbone(i % N_PROT, L_RES) for i in range(threads)]

    def one(i):
        c, s = inputs[i]
        ref.design(c, s, seqs_per_thread, seed=1000 + i, temperature=TEMP, decode_order=0,
                   keep_log_probs=True)

    t0 = time.perf_counter()
    with ThreadPoolExecutor(max_workers=threads) as ex:
        list(ex.map(one, range(threads)))
    dt = time.perf_counter() - t0
    res = threads * seqs_per_thread * L_RES
    desc = (f"{threads} threads x {seqs_per_thread} seq of L=256 (config-2 backbones, T=0.1, "
            f"random order) through the reference design path: {res} residues in {dt:.2f} s")
    return res / dt, desc


def host_cores():
    try:
        return len(os.sched_getaffinity(0))
    except AttributeError:
        return os.cpu_count() or 1


def run_reference(args):
    rank, world, _ = dist_env()
    if rank != 0:
        return 0
    cores = host_cores()
    for _ in range(args.warmup):
        cpu_baseline_sample(cores)
    vals = []
    t0 = time.perf_counter()
    desc = ""
    for _ in range(args.steps):
        v, desc = cpu_baseline_sample(cores)
        vals.append(v)
    wall = time.perf_counter() - t0
    value = float(np.mean(vals))
    line = {
        "impl": "reference", "metric": METRIC, "value": value, "unit": "residues/s",
        "n_gpus": world, "steps": args.steps, "warmup": args.warmup,
        "ms_per_step": wall * 1000 / max(1, args.steps), "higher_is_better": True,
        "scaling": "weak", "vs_baseline": None, "dtype": "f32", "data": "synthetic",
        "config": {"workload": "config2 sample: bounded per-step sample of 64 x L256 x 32 "
                               "seqs design, T=0.1, random order",
                   "proteins": N_PROT, "residue_count": L_RES, "seqs_per_protein": N_SEQ},
        "cpu_baseline": {"value": value, "unit": "residues/s", "cores": cores,
                         "kind": "reference", "sample": desc},
        "e2e": {"value": value, "unit": "residues/s", "h2d_bytes_per_step": 0,
                "d2h_bytes_per_step": 0},
    }
    print(json.dumps(line), flush=True)
    return 0


def run_ours(args):
    import torch
    rank, world, local = dist_env()
    torch.cuda.set_device(local)
    dev = torch.device("cuda", local)
    if world > 1:
        import datetime
        import torch.distributed as dist
        dist.init_process_group("nccl", timeout=datetime.timedelta(seconds=120),
                                device_id=dev)
    from hikoboshi_b200 import DesignEngine
    from hikoboshi_b200 import _lib as hl

    eng = DesignEngine(engine_weights(), device=local, precision=args.precision)
    coords_h, src_h = make_inputs(rank)
    R = coords_h.shape[0]
    Q = N_PROT * N_SEQ * L_RES
    NS = N_PROT * N_SEQ
    L = np.full(N_PROT, L_RES, np.int32)
    S = np.full(N_PROT, N_SEQ, np.int32)
    seeds = (np.arange(N_PROT, dtype=np.uint64) + np.uint64(rank * N_PROT)) * np.uint64(1000)
    temps = np.full(N_PROT, TEMP, np.float32)
    modes = np.zeros(N_PROT, np.int32)
    P = ctypes.POINTER

    def batch(cp, sp):
        return hl.DesignBatch(N_PROT, L.ctypes.data_as(P(ctypes.c_int32)), cp, sp,
                              S.ctypes.data_as(P(ctypes.c_int32)),
                              seeds.ctypes.data_as(P(ctypes.c_uint64)),
                              temps.ctypes.data_as(P(ctypes.c_float)),
                              modes.ctypes.data_as(P(ctypes.c_int32)), None)

    # device-resident inputs and outputs
    d_coords = torch.from_numpy(coords_h).to(dev)
    d_src = torch.from_numpy(src_h).to(dev)
    d_tok = torch.empty(Q, dtype=torch.int32, device=dev)
    d_lp = torch.empty(Q * 21, dtype=torch.float32, device=dev)
    d_ord = torch.empty(Q, dtype=torch.int32, device=dev)
    d_sc = torch.empty(NS, dtype=torch.float32, device=dev)
    bdev = batch(ctypes.c_void_p(d_coords.data_ptr()), ctypes.c_void_p(d_src.data_ptr()))
    odev = hl.DesignOut(ctypes.c_void_p(d_tok.data_ptr()), ctypes.c_void_p(d_lp.data_ptr()),
                        ctypes.c_void_p(d_ord.data_ptr()), ctypes.c_void_p(d_sc.data_ptr()))
    # A dedicated stream: the engine launches on it, the events time it.
    stream = torch.cuda.Stream(dev)
    torch.cuda.set_stream(stream)
    flush = torch.empty(128 * 1024 * 1024, dtype=torch.float32, device=dev)  # 512 MiB

    def device_step():
        st = hl.load().hkb_mpnn_design_device(eng._h, ctypes.byref(bdev), ctypes.byref(odev),
                                              ctypes.c_void_p(stream.cuda_stream))
        hl.check(st)

    def barrier():
        if world > 1:
            import torch.distributed as dist
            dist.barrier()
        torch.cuda.synchronize(dev)

    for _ in range(max(3, args.warmup)):
        flush.zero_()
        device_step()
    barrier()

    clocks = ClockSampler(local)
    clocks.start()
    step_ms, decode_ms, launches = [], [], 0
    t_wall0 = time.perf_counter()
    for _ in range(args.steps):
        flush.zero_()
        e0 = torch.cuda.Event(enable_timing=True)
        e1 = torch.cuda.Event(enable_timing=True)
        e0.record(stream)
        device_step()
        e1.record(stream)
        e1.synchronize()
        step_ms.append(e0.elapsed_time(e1))
        decode_ms.append(eng.last_timings()["decode_ms"])
        launches += eng.last_launch_count()
    barrier()
    wall_s = time.perf_counter() - t_wall0
    clk = clocks.stop()

    # end-to-end through the host API, pinned host buffers
    pin_c = torch.from_numpy(coords_h).pin_memory()
    pin_s = torch.from_numpy(src_h).pin_memory()
    h_tok = torch.empty(Q, dtype=torch.int32).pin_memory()
    h_lp = torch.empty(Q * 21, dtype=torch.float32).pin_memory()
    h_sc = torch.empty(NS, dtype=torch.float32).pin_memory()
    bh = batch(ctypes.c_void_p(pin_c.data_ptr()), ctypes.c_void_p(pin_s.data_ptr()))
    oh = hl.DesignOut(ctypes.c_void_p(h_tok.data_ptr()), ctypes.c_void_p(h_lp.data_ptr()),
                      None, ctypes.c_void_p(h_sc.data_ptr()))

    def host_step():
        hl.check(hl.load().hkb_mpnn_design(eng._h, ctypes.byref(bh), ctypes.byref(oh)))

    host_step()
    barrier()
    e2e_steps = max(1, min(args.steps, 5))
    t0 = time.perf_counter()
    for _ in range(e2e_steps):
        host_step()
    e2e_s = (time.perf_counter() - t0) / e2e_steps
    barrier()

    step_s = float(np.mean(step_ms)) / 1000.0
    dec_s = float(np.mean(decode_ms)) / 1000.0
    stats = torch.tensor([step_s, dec_s, e2e_s], dtype=torch.float64, device=dev)
    if world > 1:
        import torch.distributed as dist
        dist.all_reduce(stats, op=dist.ReduceOp.MAX)
    step_s, dec_s, e2e_s = stats.tolist()

    if rank == 0:
        res_step = Q * world
        value = res_step / step_s
        peaks, kind = measured_peaks()
        peak = peaks["bf16_tflops"]
        achieved = FLOP_DECODE_PER_RES * Q / dec_s / 1e12
        traffic = profiled_traffic(args.precision)
        line = {
            "metric": METRIC, "value": value, "unit": "residues/s", "n_gpus": world,
            "steps": args.steps, "warmup": max(3, args.warmup), "ms_per_step": step_s * 1000,
            "higher_is_better": True, "scaling": "weak", "vs_baseline": None,
            "dtype": {"f16": "f16", "bf16": "bf16", "fp32": "f32"}[args.precision],
            "data": data_note("synthetic (seeded ideal-geometry backbones, BASELINE generator)"),
            "config": {"workload": "config2: 64 backbones x L=256 x 32 seqs per GPU, T=0.1, "
                                   "random decoding order per sequence",
                       "proteins_per_gpu": N_PROT, "residue_count": L_RES,
                       "seqs_per_protein": N_SEQ, "temperature": TEMP,
                       "precision": args.precision,
                       "l2": "flushed before every step (512 MiB write, outside the events)"},
            "us_per_decode_step": dec_s / L_RES * 1e6,
            "decode_ms": dec_s * 1000,
            "roofline": {"bound": "tensor", "kernel": "ar_decode",
                         "achieved": achieved, "peak": peak, "unit": "TFLOP/s",
                         "frac": achieved / peak, "traffic": traffic,
                         "flops_per_launch": FLOP_DECODE_PER_RES * Q,
                         "peak_kind": f"{kind} dense 16-bit tensor burst"},
            "e2e": {"value": res_step / e2e_s, "unit": "residues/s",
                    "h2d_bytes_per_step": int(coords_h.nbytes + src_h.nbytes),
                    "d2h_bytes_per_step": int(Q * 4 + Q * 21 * 4 + NS * 4)},
            "gpu_launches": int(launches / max(1, args.steps)),
            "gpu_launches_total": int(launches),
            "clocks": clk,
            "wall_s": wall_s,
        }
        if not args.no_cpu_baseline:
            cores = host_cores()
            v, desc = cpu_baseline_sample(cores)
            line["cpu_baseline"] = {"value": v, "unit": "residues/s", "cores": cores,
                                    "kind": "reference", "sample": desc}
        print(json.dumps(line), flush=True)
    eng.close()
    if world > 1:
        import torch.distributed as dist
        dist.barrier()
        dist.destroy_process_group()
    return 0


# ---------------------------------------------------------------------------
# teacher-forced scoring, 128 x L=384 x 16 random sequences
# ---------------------------------------------------------------------------
C4_PROT, C4_L, C4_SEQ = 128, 384, 16
METRIC4 = "ProteinMPNN v48 teacher-forced scored residues/sec at 128 x L=384 x 16 seqs"


def config4_inputs(rank: int, synth):
    """Backbone i of rank r: generator seed 3000 + 128 r + i; tokens uniform
    over the 20 amino acids from numpy's default_rng(3 + r); random decoding
    order per sequence from seed 3 + s."""
    bb = [synth(3000 + C4_PROT * rank + i, C4_L) for i in range(C4_PROT)]
    rng = np.random.default_rng(3 + rank)
    toks = [rng.integers(0, 20, (C4_SEQ, C4_L)).astype(np.int32) for _ in range(C4_PROT)]
    return [b[0] for b in bb], [b[1] for b in bb], toks


def cpu_baseline_config4(threads: int):
    """The reference's teacher-forced forward (compiled from its sources), one
    config-4 sequence per host thread."""
    from concurrent.futures import ThreadPoolExecutor
    from oracle.oracle import RefLib
    ref = RefLib(WEIGHTS)
    cs, ss, toks = config4_inputs(0, ref.synthetic_backbone)

    def one(i):
        b = i % C4_PROT
        ref.teacher_forced(cs[b], ss[b], toks[b][i % C4_SEQ], None, seed=3 + i % C4_SEQ)

    t0 = time.perf_counter()
    with ThreadPoolExecutor(max_workers=threads) as ex:
        list(ex.map(one, range(threads)))
    dt = time.perf_counter() - t0
    res = threads * C4_L
    desc = (f"{threads} threads x 1 sequence of L=384 (config-4 backbones and tokens, random "
            f"order) through the reference teacher-forced forward: {res} residues in {dt:.2f} s")
    return res / dt, desc


def run_config4(args):
    import torch
    rank, world, local = dist_env()
    torch.cuda.set_device(local)
    dev = torch.device("cuda", local)
    if args.impl == "reference":
        if rank != 0:
            return 0
        cores = host_cores()
        for _ in range(args.warmup):
            cpu_baseline_config4(cores)
        vals, desc = [], ""
        t0 = time.perf_counter()
        for _ in range(args.steps):
            v, desc = cpu_baseline_config4(cores)
            vals.append(v)
        value = float(np.mean(vals))
        print(json.dumps({
            "impl": "reference", "metric": METRIC4, "value": value, "unit": "residues/s",
            "n_gpus": world, "steps": args.steps, "warmup": args.warmup,
            "ms_per_step": (time.perf_counter() - t0) * 1000 / max(1, args.steps),
            "higher_is_better": True, "scaling": "weak", "vs_baseline": None, "dtype": "f32",
            "data": "synthetic", "config": {"workload": "config4 sample"},
            "cpu_baseline": {"value": value, "unit": "residues/s", "cores": cores,
                             "kind": "reference", "sample": desc},
            "e2e": {"value": value, "unit": "residues/s", "h2d_bytes_per_step": 0,
                    "d2h_bytes_per_step": 0}}), flush=True)
        return 0
    if world > 1:
        import datetime
        import torch.distributed as dist
        dist.init_process_group("nccl", timeout=datetime.timedelta(seconds=120), device_id=dev)
    from hikoboshi_b200 import DesignEngine, synthetic_backbone
    eng = DesignEngine(engine_weights(), device=local, precision=args.precision)
    cs, ss, toks = config4_inputs(rank, synthetic_backbone)
    Q = C4_PROT * C4_SEQ * C4_L
    flush = torch.empty(128 * 1024 * 1024, dtype=torch.float32, device=dev)

    def barrier():
        if world > 1:
            import torch.distributed as dist
            dist.barrier()
        torch.cuda.synchronize(dev)

    def step():
        eng.score(cs, ss, toks, seeds=3)

    for _ in range(max(3, args.warmup)):
        flush.zero_()
        torch.cuda.synchronize(dev)
        step()
    barrier()
    clocks = ClockSampler(local)
    clocks.start()
    dev_ms, tf_ms, launches = [], [], 0
    for _ in range(args.steps):
        flush.zero_()
        torch.cuda.synchronize(dev)
        step()
        tm = eng.last_timings()
        dev_ms.append(tm["total_ms"])
        tf_ms.append(tm["decode_ms"])
        launches += eng.last_launch_count()
    barrier()
    clk = clocks.stop()

    # end-to-end through the host API (hkb_mpnn_score) with pinned host
    # buffers: coordinates, atom sources and tokens uploaded, log-probs,
    # orders and scores read back every call
    import hikoboshi_b200._lib as hl
    P = ctypes.POINTER
    L = np.full(C4_PROT, C4_L, np.int32)
    S = np.full(C4_PROT, C4_SEQ, np.int32)
    seeds = np.full(C4_PROT, 3, np.uint64)
    pin_c = torch.from_numpy(np.ascontiguousarray(np.concatenate(cs), np.float32)).pin_memory()
    pin_s = torch.from_numpy(np.ascontiguousarray(np.concatenate(ss), np.uint8)).pin_memory()
    pin_t = torch.from_numpy(np.ascontiguousarray(np.concatenate([t.reshape(-1) for t in toks]),
                                                  np.int32)).pin_memory()
    h_lp = torch.empty(Q * 21, dtype=torch.float32).pin_memory()
    h_ord = torch.empty(Q, dtype=torch.int32).pin_memory()
    h_sc = torch.empty(C4_PROT * C4_SEQ, dtype=torch.float32).pin_memory()
    sb = hl.ScoreBatch(C4_PROT, L.ctypes.data_as(P(ctypes.c_int32)),
                       ctypes.c_void_p(pin_c.data_ptr()), ctypes.c_void_p(pin_s.data_ptr()),
                       S.ctypes.data_as(P(ctypes.c_int32)),
                       ctypes.cast(ctypes.c_void_p(pin_t.data_ptr()), P(ctypes.c_int32)),
                       None, seeds.ctypes.data_as(P(ctypes.c_uint64)))
    so = hl.ScoreOut(ctypes.c_void_p(h_lp.data_ptr()), ctypes.c_void_p(h_ord.data_ptr()),
                     ctypes.c_void_p(h_sc.data_ptr()))

    def host_step():
        hl.check(hl.load().hkb_mpnn_score(eng._h, ctypes.byref(sb), ctypes.byref(so)))

    host_step()
    barrier()
    wall_ms = []
    for _ in range(max(1, min(args.steps, 5))):
        t0 = time.perf_counter()
        host_step()
        wall_ms.append((time.perf_counter() - t0) * 1000)
    barrier()
    stats = torch.tensor([np.mean(dev_ms), np.mean(tf_ms), np.mean(wall_ms)], dtype=torch.float64,
                         device=dev)
    if world > 1:
        import torch.distributed as dist
        dist.all_reduce(stats, op=dist.ReduceOp.MAX)
    d_ms, t_ms, w_ms = stats.tolist()
    if rank == 0:
        peaks, kind = measured_peaks()
        achieved = FLOP_DECODE_PER_RES * Q / (t_ms / 1000) / 1e12
        line = {
            "metric": METRIC4, "value": Q * world / (d_ms / 1000), "unit": "residues/s",
            "n_gpus": world, "steps": args.steps, "warmup": max(3, args.warmup),
            "ms_per_step": d_ms, "higher_is_better": True, "scaling": "weak",
            "vs_baseline": None, "dtype": {"f16": "f16", "bf16": "bf16", "fp32": "f32"}[args.precision],
            "data": data_note("synthetic (seeded ideal-geometry backbones, uniform random "
                              "tokens)"),
            "config": {"workload": "config4: teacher-forced scoring of 128 backbones x L=384 x 16 "
                                   "sequences per GPU, random decoding order",
                       "precision": args.precision,
                       "l2": "flushed before every step (512 MiB write, outside the timing)",
                       "timing": "value: device events around the pipeline (encoder, tables, "
                                 "teacher-forced layers); e2e: the host call (hkb_mpnn_score) "
                                 "from pinned buffers with uploads and log-prob read-back"},
            "tf_ms": t_ms,
            "roofline": {"bound": "tensor", "kernel": "teacher-forced layers (tf_slot_tc + tf_node_tc)",
                         "achieved": achieved, "peak": peaks["bf16_tflops"], "unit": "TFLOP/s",
                         "frac": achieved / peaks["bf16_tflops"], "traffic": None,
                         "flops_per_launch": FLOP_DECODE_PER_RES * Q,
                         "peak_kind": f"{kind} dense 16-bit tensor burst"},
            "e2e": {"value": Q * world / (w_ms / 1000), "unit": "residues/s",
                    "h2d_bytes_per_step": int(C4_PROT * C4_L * 20 + Q * 4),
                    "d2h_bytes_per_step": int(Q * 21 * 4 + Q * 4 + C4_PROT * C4_SEQ * 4)},
            "gpu_launches": int(launches / max(1, args.steps)),
            "clocks": clk,
        }
        if not args.no_cpu_baseline:
            cores = host_cores()
            v, desc = cpu_baseline_config4(cores)
            line["cpu_baseline"] = {"value": v, "unit": "residues/s", "cores": cores,
                                    "kind": "reference", "sample": desc}
        print(json.dumps(line), flush=True)
    eng.close()
    if world > 1:
        import torch.distributed as dist
        dist.barrier()
        dist.destroy_process_group()
    return 0


# ---------------------------------------------------------------------------
# box-wide sweep, 4096 backbones L ~ U[64, 512] x 16 seqs
# ---------------------------------------------------------------------------
C5_PROT, C5_SEQ = 4096, 16
METRIC5 = "ProteinMPNN v48 designed residues/sec box-wide, 4096 backbones L~U[64,512] x16 seqs"
C5_CHUNK_RES = 4_194_304    # designed residues per device call (bounds device memory)


def config5_lengths():
    return [int(x) for x in np.random.default_rng(42).integers(64, 513, C5_PROT)]


def config5_backbone(i: int, L: int, synth):
    return synth(42_000 + i, L)


def cpu_baseline_config5(threads: int):
    """Stratified sample: one sequence per host thread, lengths at evenly
    spaced quantiles of the config-5 length list; per-residue throughput of
    the reference design path (the box-wide figure extrapolates it)."""
    from concurrent.futures import ThreadPoolExecutor
    from oracle.oracle import RefLib
    ref = RefLib(WEIGHTS)
    Ls = config5_lengths()
    order = np.argsort(Ls, kind="stable")
    pick = [int(order[int((k + 0.5) * C5_PROT / threads)]) for k in range(threads)]
    inputs = [config5_backbone(i, Ls[i], ref.synthetic_backbone) for i in pick]

    def one(k):
        c, s = inputs[k]
        ref.design(c, s, 1, seed=pick[k], temperature=TEMP, decode_order=0, keep_log_probs=False)

    t0 = time.perf_counter()
    with ThreadPoolExecutor(max_workers=threads) as ex:
        list(ex.map(one, range(threads)))
    dt = time.perf_counter() - t0
    res = sum(Ls[i] for i in pick)
    desc = (f"stratified sample: {threads} threads x 1 sequence, lengths at {threads} quantiles "
            f"of the config-5 lengths ({res} residues in {dt:.2f} s); the box-wide value "
            f"extrapolates this per-residue rate")
    return res / dt, desc


def run_config5(args):
    import torch
    rank, world, local = dist_env()
    if args.impl == "reference":
        if rank != 0:
            return 0
        cores = host_cores()
        for _ in range(args.warmup):
            cpu_baseline_config5(cores)
        vals, desc = [], ""
        t0 = time.perf_counter()
        for _ in range(args.steps):
            v, desc = cpu_baseline_config5(cores)
            vals.append(v)
        value = float(np.mean(vals))
        print(json.dumps({
            "impl": "reference", "metric": METRIC5, "value": value, "unit": "residues/s",
            "n_gpus": world, "steps": args.steps, "warmup": args.warmup,
            "ms_per_step": (time.perf_counter() - t0) * 1000 / max(1, args.steps),
            "higher_is_better": True, "scaling": "strong", "vs_baseline": None, "dtype": "f32",
            "data": "synthetic", "config": {"workload": "config5 stratified sample"},
            "cpu_baseline": {"value": value, "unit": "residues/s", "cores": cores,
                             "kind": "reference", "sample": desc},
            "e2e": {"value": value, "unit": "residues/s", "h2d_bytes_per_step": 0,
                    "d2h_bytes_per_step": 0}}), flush=True)
        return 0
    torch.cuda.set_device(local)
    dev = torch.device("cuda", local)
    import datetime
    import torch.distributed as dist
    if world > 1:
        dist.init_process_group("nccl", timeout=datetime.timedelta(seconds=300), device_id=dev)
    from hikoboshi_b200 import DesignEngine, synthetic_backbone
    from hikoboshi_b200 import _lib as hl
    from hikoboshi_b200.shard import design_sharded, partition_proteins
    eng = DesignEngine(engine_weights(), device=local, precision=args.precision)
    Ls = config5_lengths()
    mine = partition_proteins(Ls, C5_SEQ, world)[rank]
    total_res = sum(Ls) * C5_SEQ
    # device-resident inputs of this rank's proteins, in chunks of whole proteins
    chunks, cur, cur_res = [], [], 0
    for b in mine:
        if cur and cur_res + Ls[b] * C5_SEQ > C5_CHUNK_RES:
            chunks.append(cur)
            cur, cur_res = [], 0
        cur.append(b)
        cur_res += Ls[b] * C5_SEQ
    if cur:
        chunks.append(cur)
    P = ctypes.POINTER
    calls = []
    max_q = max((sum(Ls[b] for b in ch) * C5_SEQ for ch in chunks), default=1)
    d_tok = torch.empty(max_q, dtype=torch.int32, device=dev)
    d_lp = torch.empty(max_q * 21, dtype=torch.float32, device=dev)
    d_ord = torch.empty(max_q, dtype=torch.int32, device=dev)
    d_sc = torch.empty(max(1, max_q // 64), dtype=torch.float32, device=dev)
    keep = []
    for ch in chunks:
        bb = [config5_backbone(b, Ls[b], synthetic_backbone) for b in ch]
        dc = torch.from_numpy(np.concatenate([x[0] for x in bb])).to(dev)
        ds = torch.from_numpy(np.concatenate([x[1] for x in bb])).to(dev)
        L = np.array([Ls[b] for b in ch], np.int32)
        S = np.full(len(ch), C5_SEQ, np.int32)
        seeds = np.array(ch, np.uint64)
        temps = np.full(len(ch), TEMP, np.float32)
        modes = np.zeros(len(ch), np.int32)
        keep += [dc, ds, L, S, seeds, temps, modes]
        calls.append(hl.DesignBatch(len(ch), L.ctypes.data_as(P(ctypes.c_int32)),
                                    ctypes.c_void_p(dc.data_ptr()), ctypes.c_void_p(ds.data_ptr()),
                                    S.ctypes.data_as(P(ctypes.c_int32)),
                                    seeds.ctypes.data_as(P(ctypes.c_uint64)),
                                    temps.ctypes.data_as(P(ctypes.c_float)),
                                    modes.ctypes.data_as(P(ctypes.c_int32)), None))
    odev = hl.DesignOut(ctypes.c_void_p(d_tok.data_ptr()), ctypes.c_void_p(d_lp.data_ptr()),
                        ctypes.c_void_p(d_ord.data_ptr()), ctypes.c_void_p(d_sc.data_ptr()))
    stream = torch.cuda.Stream(dev)
    torch.cuda.set_stream(stream)
    flush = torch.empty(128 * 1024 * 1024, dtype=torch.float32, device=dev)

    def device_step():
        for bt in calls:
            hl.check(hl.load().hkb_mpnn_design_device(eng._h, ctypes.byref(bt), ctypes.byref(odev),
                                                      ctypes.c_void_p(stream.cuda_stream)))

    def barrier():
        if world > 1:
            dist.barrier()
        torch.cuda.synchronize(dev)

    steps = max(1, args.steps)
    for _ in range(max(3, args.warmup)):
        flush.zero_()
        device_step()
    barrier()
    clocks = ClockSampler(local)
    clocks.start()
    step_ms = []
    for _ in range(steps):
        flush.zero_()
        e0 = torch.cuda.Event(enable_timing=True)
        e1 = torch.cuda.Event(enable_timing=True)
        e0.record(stream)
        device_step()
        e1.record(stream)
        e1.synchronize()
        step_ms.append(e0.elapsed_time(e1))
    barrier()
    clk = clocks.stop()
    # end to end: the sharded host API (every rank passes the whole batch,
    # designs its partition, rank 0 gathers tokens, orders and scores)
    allbb = [config5_backbone(b, Ls[b], synthetic_backbone) for b in range(C5_PROT)]
    coords, sources = [x[0] for x in allbb], [x[1] for x in allbb]

    def host_step():
        return design_sharded(eng, coords, sources, C5_SEQ, seeds=list(range(C5_PROT)),
                              temperatures=TEMP, keep_log_probs=False,
                              max_rows_per_call=C5_CHUNK_RES)

    host_step()
    barrier()
    e2e_steps = max(1, min(steps, 3))
    t0 = time.perf_counter()
    for _ in range(e2e_steps):
        host_step()
    barrier()
    e2e_s = (time.perf_counter() - t0) / e2e_steps
    stats = torch.tensor([float(np.mean(step_ms))], dtype=torch.float64, device=dev)
    if world > 1:
        dist.all_reduce(stats, op=dist.ReduceOp.MAX)
    step_s = stats.item() / 1000
    if rank == 0:
        peaks, kind = measured_peaks()
        flops = FLOP_DECODE_PER_RES * total_res + FLOP_ENCODE_PER_RES * sum(Ls)
        achieved = flops / step_s / 1e12
        line = {
            "metric": METRIC5, "value": total_res / step_s, "unit": "residues/s",
            "n_gpus": world, "steps": steps, "warmup": max(3, args.warmup),
            "ms_per_step": step_s * 1000, "higher_is_better": True, "scaling": "strong",
            "vs_baseline": None, "dtype": {"f16": "f16", "bf16": "bf16", "fp32": "f32"}[args.precision],
            "data": data_note("synthetic (seeded ideal-geometry backbones, lengths from "
                              "default_rng(42))"),
            "config": {"workload": "config5: 4096 backbones, L uniform in [64, 512], 16 seqs each, "
                                   "T=0.1, length-bucketed LPT partition by protein over the ranks",
                       "designed_residues": total_res, "precision": args.precision,
                       "l2": "flushed before every step (512 MiB write)",
                       "device_calls_per_rank": len(calls)},
            "per_gpu_residues_per_s": total_res / step_s / world,
            "roofline": {"bound": "tensor", "kernel": "whole design step (encoder + decode)",
                         "achieved": achieved, "peak": peaks["bf16_tflops"] * world,
                         "unit": "TFLOP/s", "frac": achieved / (peaks["bf16_tflops"] * world),
                         "traffic": None, "flops_per_launch": flops,
                         "peak_kind": f"{kind} dense 16-bit tensor burst x {world} GPUs"},
            "e2e": {"value": total_res / e2e_s, "unit": "residues/s",
                    "h2d_bytes_per_step": int(sum(Ls) * 80),
                    "d2h_bytes_per_step": int(total_res * 8 + C5_PROT * C5_SEQ * 4)},
            "clocks": clk,
        }
        if not args.no_cpu_baseline:
            cores = host_cores()
            v, desc = cpu_baseline_config5(cores)
            line["cpu_baseline"] = {"value": v, "unit": "residues/s", "cores": cores,
                                    "kind": "reference", "sample": desc}
        print(json.dumps(line), flush=True)
    eng.close()
    if world > 1:
        dist.barrier()
        dist.destroy_process_group()
    return 0


# ---------------------------------------------------------------------------
# BASELINE configs 1 and 3 (parity cases), timed on both arms for the record
# ---------------------------------------------------------------------------
SMALL = {"config1": dict(L=128, seed=7, S=8, T=0.1, ref_seqs=8,
                         desc="1 backbone L=128 (seed 7) x 8 sequences, T=0.1"),
         "config3": dict(L=1024, seed=11, S=256, T=0.2, ref_seqs=16,
                         desc="1 backbone L=1024 (seed 11) x 256 sequences, T=0.2")}


def run_small(args):
    """Config 1 (the reference's own CPU-runnable case) and config 3 (one long
    chain).  Ours: the host API (`design`), value from the device events of
    the call, e2e from the wall clock.  Reference: the reference design path
    on the host cores, one sequence per thread; for config 3 a 16-sequence
    subset whose per-residue rate stands for the 256-sequence run (labelled
    extrapolated)."""
    import torch
    cfg = SMALL[args.workload]
    rank, world, local = dist_env()
    if rank != 0:
        return 0
    if args.impl == "reference":
        from concurrent.futures import ThreadPoolExecutor
        from oracle.oracle import RefLib
        ref = RefLib(WEIGHTS)
        c, s_ = ref.synthetic_backbone(cfg["seed"], cfg["L"])
        n = cfg["ref_seqs"]
        cores = host_cores()

        def sample():
            t0 = time.perf_counter()
            with ThreadPoolExecutor(max_workers=min(cores, n)) as ex:
                list(ex.map(lambda q: ref.design(c, s_, 1, seed=q, temperature=cfg["T"],
                                                 decode_order=0, keep_log_probs=False), range(n)))
            return n * cfg["L"] / (time.perf_counter() - t0)

        for _ in range(args.warmup):
            sample()
        vals = [sample() for _ in range(args.steps)]
        value = float(np.mean(vals))
        desc = (f"{n} sequences of the {args.workload} backbone, one per thread on "
                f"{min(cores, n)} threads" + (" (subset of 256; per-residue rate extrapolated)"
                                              if args.workload == "config3" else ""))
        print(json.dumps({
            "impl": "reference", "metric": f"ProteinMPNN v48 designed residues/sec, {cfg['desc']}",
            "value": value, "unit": "residues/s", "n_gpus": world, "steps": args.steps,
            "warmup": args.warmup, "ms_per_step": n * cfg["L"] / value * 1000,
            "higher_is_better": True, "scaling": "weak", "vs_baseline": None, "dtype": "f32",
            "data": "synthetic", "config": {"workload": args.workload},
            "cpu_baseline": {"value": value, "unit": "residues/s", "cores": min(cores, n),
                             "kind": "reference", "sample": desc},
            "e2e": {"value": value, "unit": "residues/s", "h2d_bytes_per_step": 0,
                    "d2h_bytes_per_step": 0}}), flush=True)
        return 0
    torch.cuda.set_device(local)
    from hikoboshi_b200 import DesignEngine, synthetic_backbone
    eng = DesignEngine(engine_weights(), device=local, precision=args.precision)
    c, s_ = synthetic_backbone(cfg["seed"], cfg["L"])
    res_step = cfg["S"] * cfg["L"]
    for _ in range(max(3, args.warmup)):
        eng.design([c], [s_], num_seqs=cfg["S"], seeds=0, temperatures=cfg["T"])
    dev, wall = [], []
    for _ in range(args.steps):
        t0 = time.perf_counter()
        eng.design([c], [s_], num_seqs=cfg["S"], seeds=0, temperatures=cfg["T"])
        wall.append(time.perf_counter() - t0)
        dev.append(eng.last_timings()["total_ms"] / 1000)
    print(json.dumps({
        "metric": f"ProteinMPNN v48 designed residues/sec, {cfg['desc']}",
        "value": res_step / float(np.mean(dev)), "unit": "residues/s", "n_gpus": 1,
        "steps": args.steps, "warmup": max(3, args.warmup), "ms_per_step": float(np.mean(dev)) * 1000,
        "higher_is_better": True, "scaling": "weak", "vs_baseline": None,
        "dtype": {"f16": "f16", "bf16": "bf16", "fp32": "f32"}[args.precision],
        "data": data_note("synthetic"),
        "config": {"workload": args.workload, "precision": args.precision},
        "e2e": {"value": res_step / float(np.mean(wall)), "unit": "residues/s",
                "h2d_bytes_per_step": cfg["L"] * 80,
                "d2h_bytes_per_step": res_step * (4 + 21 * 4 + 4) + cfg["S"] * 4}}), flush=True)
    eng.close()
    return 0


def run_profile_case(args):
    """One untimed call on a small case for ncu captures: ``design`` runs
    N backbones x L=256 x S sequences (T=0.1; S = 32 by default, 128 gives
    the config-2 occupancy of 14 sequences per decode CTA on 16 backbones),
    ``score`` the teacher-forced pass over N backbones x L=384 x 16 random
    sequences (the config-2 and config-4 shapes with N proteins, default
    16)."""
    from hikoboshi_b200 import DesignEngine, synthetic_backbone
    n = args.profile_proteins
    eng = DesignEngine(engine_weights(), device=0, precision=args.precision)
    if args.profile_workload == "score":
        cs, ss, toks = config4_inputs(0, synthetic_backbone)
        eng.score(cs[:n], ss[:n], toks[:n], seeds=3)
        case = f"{n} x L=384 x 16 teacher-forced"
    else:
        bb = [synthetic_backbone(i, L_RES) for i in range(n)]
        eng.design([b[0] for b in bb], [b[1] for b in bb], num_seqs=args.profile_seqs,
                   seeds=list(range(n)), temperatures=TEMP, keep_log_probs=True)
        case = f"{n} x L=256 x {args.profile_seqs} design"
    print(json.dumps({"profile_case": case, "precision": args.precision, **eng.last_timings()}))
    eng.close()
    return 0


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=10)
    ap.add_argument("--warmup", type=int, default=3)
    ap.add_argument("--impl", choices=["ours", "reference"], default="ours")
    ap.add_argument("--precision", choices=["f16", "bf16", "fp32"], default="f16")
    ap.add_argument("--no-cpu-baseline", action="store_true")
    ap.add_argument("--workload", choices=["config1", "config2", "config3", "config4", "config5"],
                    default="config2",
                    help="config2 (default): batched design; config4: teacher-forced scoring; "
                         "config5: the mixed-length sweep sharded over the ranks")
    ap.add_argument("--profile-case", action="store_true",
                    help="one untimed call on a small case (for ncu captures)")
    ap.add_argument("--profile-workload", choices=["design", "score"], default="design")
    ap.add_argument("--profile-proteins", type=int, default=16)
    ap.add_argument("--profile-seqs", type=int, default=32)
    args = ap.parse_args()
    missing = reference_missing()
    if missing and args.impl == "reference":
        if dist_env()[0] == 0:
            print(json.dumps({"impl": "reference", "unavailable": missing}), flush=True)
        return 0
    if missing:
        args.no_cpu_baseline = True
    if args.profile_case:
        return run_profile_case(args)
    if args.workload in SMALL:
        return run_small(args)
    if args.workload == "config4":
        return run_config4(args)
    if args.workload == "config5":
        return run_config5(args)
    if args.impl == "reference":
        return run_reference(args)
    return run_ours(args)


if __name__ == "__main__":
    sys.exit(main())
