#!/usr/bin/env python
"""Headline benchmark: rendered rays/sec (fwd+bwd) at 512x512, 64(+2+32 extra) samples per fg node after
the 128-sample error-bound hierarchy, single-hand scene (right hand + object + background).

One "step" (default --mode train) = zero the gradient bucket + one full forward + Loss + backward pass of the HIP hot
path over one synthetic 512x512 frame (262 144 rays) per GPU, ray-chunked with gradient accumulation + the optimiser
step (hold_amd.optim.FlatAdam: RCCL all-reduce of the flat gradient bucket when N > 1, global-norm clip, Adam).
Inputs (rays, poses, weights, gt) are resident in HBM before the timed region.

    python bench.py --gpus 1 --steps 2 --warmup 1
    python -m torch.distributed.run --nnodes=1 --nproc-per-node N ... bench.py --gpus N --steps K --warmup W

Other workloads of BASELINE.json (secondary lines, same JSON contract):
    --mode render            C2 eval-mode forward only
    --two-hands              C4-like ARCTIC scene (right + left + object)
    --mode c3                C3: the reference's own training step (10 frames x 128 rays, full Loss, pose-table
                             gradients, Adam) in steps/s -> value is still rays/s; plus pose-refinement iters/s
    --mode c5                C5: 1024x1024 eval render with N_samples = 128 (162 samples per fg node)
    --loss pixel|full        train modes: rgb + semantic loss only (what round 1 timed) or the full reference Loss
                             with the canonical-mesh loss targets (eikonal, MANO-cano SDF, opacity sparsity)
    --fp32-mfma              every matrix product on the fp32 MFMA (default: the sampler trunk and the weight-gradient
                             kernel use the exact 3-limb bf16 split, see hold_amd/config.py)

Prints ONE JSON line (rank 0) with the driver's contract fields plus `roofline` (the MFMA kernel with the largest share
of the timed region, measured live with events on the launch stream; every kernel's figures under roofline.kernels)
and `cpu_baseline` (the CPU oracle restatement of the reference timed on this box's host cores).
"""
import argparse
import json
import os
import sys
import time

import numpy as np
import torch

ROOT = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, ROOT)

FP32_MFMA_PEAK_TFLOPS = 157.3  # /opt/skills/guides/MI355X_MICROARCH.md (dense fp32 matrix)
BF16_MFMA_PEAK_TFLOPS = 2500.0  # dense bf16 matrix, same guide
HBM_PEAK_GBPS = 8000.0  # HBM3E spec (6.3 TB/s achievable by a float4 copy), same guide
ROUND = "r06"


def parse():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=2)
    ap.add_argument("--warmup", type=int, default=1)
    ap.add_argument("--res", type=int, default=None, help="frame side (default 512; 1024 for --mode c5)")
    ap.add_argument("--chunk", type=int, default=16384, help="rays per microbatch (~85 GB of saved activations per fg node)")
    ap.add_argument("--no-cpu-baseline", action="store_true")
    ap.add_argument("--cpu-threads", type=int, default=32)
    ap.add_argument("--cpu-frames", type=int, default=1, help="frames (x 128 rays) of the reference's 10-frame step the cpu_baseline leg times")
    ap.add_argument("--mode", default="train", choices=["train", "render", "c3", "c5"])
    ap.add_argument("--loss", default="full", choices=["pixel", "full"])
    ap.add_argument("--two-hands", action="store_true", help="ARCTIC-style scene (right + left + object), config C4")
    ap.add_argument("--fp32-mfma", action="store_true", help="true-fp32 MFMA everywhere (no split-precision kernels)")
    ap.add_argument("--beta", type=float, default=None,
                    help="Laplace density beta of the foreground nodes (default: the synthetic scene's 0.1, the reference's "
                         "INITIAL value, density.py:21-30; a trained HOLD model has beta ~ 0.005: sdf -> density is then an exact "
                         "fp32 zero half a scene unit off the surface and exact sample compaction has something to drop)")
    ap.add_argument("--no-compact", action="store_true",
                    help="A/B: run every sample through every stage (hold_amd.field.COMPACT = False)")
    ap.add_argument("--precision", default=None, choices=["f32", "f32x6", "f16x3"],
                    help="arithmetic of the MFMA kernels (hold_amd/config.py); default: the package default")
    ap.add_argument("--optimizer", default="adam", choices=["adam", "muon"],
                    help="adam: the reference's; muon: hidden matrices by orthogonalised momentum (hold_amd.optim.FlatMuon)")
    ap.add_argument("--no-profile", action="store_true")
    ap.add_argument("--c2-alt", action="store_true",
                    help="SURVEY 8(d)'s second reading of BASELINE's '64+64 samples': N_samples_eval=64 coarse + N_samples=64 fine, no extras "
                         "(66 z per node instead of 128 -> 98) -- a secondary line")
    ap.add_argument("--op-sites", default=None, metavar="PATH",
                    help="diagnostic: count the non-view torch operators of ONE extra step by the hold_amd source line that "
                         "issued them (TorchDispatchMode; run after the timed steps) and write the table to PATH")
    ap.add_argument("--step-times", default=None, metavar="PATH",
                    help="diagnostic: after the timed steps run 16 more, each timed on its own with a synchronisation, and write the "
                         "times with the caching allocator's counters to PATH")
    ap.add_argument("--sync-debug", default=None, metavar="PATH",
                    help="diagnostic: write the call sites of every host<->device synchronisation of the timed steps to PATH")
    ap.add_argument("--torch-profile", default=None, metavar="PATH",
                    help="diagnostic: run the timed steps under torch.profiler and write the per-operator call counts / "
                         "host and device times to PATH (the step time of such a run is perturbed; not a bench line)")
    ap.add_argument("--cprofile", default=None, metavar="PATH",
                    help="diagnostic: the host's Python time of the timed steps by function (cProfile on the main thread and, "
                         "through wrapped autograd Function.backward bodies, on the autograd engine's thread) -> PATH")
    ap.add_argument("--no-refine", action="store_true", help="--mode c3: skip the pose-refinement leg")
    ap.add_argument("--c3-pixels", type=int, default=128,
                    help="--mode c3: random pixels per frame (the reference's num_sample, general.yaml:82: 128 -> 1 280 rays per step; "
                         "larger values show the 10-frame step device-bound -- a secondary line, labelled in config.workload)")
    ap.add_argument("--no-freeze", action="store_true",
                    help="let Adam move the weights during the run (default: the flat parameter bucket is restored after "
                         "every optimiser step, inside the timed region, so that every step sees the same SDF and runs the "
                         "same number of sampler rounds -- the workload of step 1 is the workload of step K)")
    ap.add_argument("--split", default="frames", choices=["frames", "rays"],
                    help="multi-GPU partition: 'frames' = one frame per rank (weak scaling, the default); 'rays' = ONE frame, "
                         "contiguous ray tiles per rank, the sampler's convergence test synchronised by a 2-float MAX all-reduce "
                         "per round (strong scaling, SURVEY 8(e))")
    ap.add_argument("--shape-report", default="", help="write per-(kernel, flop bucket) launch aggregates to this json file")
    return ap.parse_args()


def cpu_baseline(sc, sd_np, threads=32, repeats=3, n_frames=1):
    """The CPU oracle (torch restatement of the reference's PyTorch path, oracle/hold_oracle.py + oracle/targets_oracle.py)
    timed on the host in the REFERENCE'S OWN step shape: 10 frames x 128 random pixels = 1 280 rays
    (general.yaml:82, tempo_dataset.py:27-36), forward + the loss targets of a steady-state step (off-surface test of every
    canonical sample against the node's loss-target mesh, MANO-canonical SDF and eikonal samples, hold_utils.py:149-240) +
    the full Loss (code/src/hold/loss.py:17-93) + backward.  BOUNDED SAMPLE: `n_frames` of the step's 10 frames (default 1 =
    128 rays; every term is a sum over frames / rays, the cost is linear in them: `--cpu-frames 10` times the whole 1 280-ray
    step, 114 s on round 4's GPU box), ONE untimed warm-up of the network part, then `repeats` (>= 3, BASELINE.md section 3:
    median of repeated steps) timed steps with fresh pixel draws; median and spread are reported.  Each step is timed in TWO
    parts: `network` = forward + Loss + backward (every repeat), and `loss_target_geometry` = the exact
    point-to-mesh distances of the loss targets, 1.2e6 point-triangle tests per ray on the host (98 % of the step, deterministic
    arithmetic: timed in the FIRST repeat only, on every 4th ray with the time scaled by 4 -- the cost is exactly linear in the points,
    and in full it is 60-100 s per 128 rays on the pool's hosts -- so that the default bench run stays within minutes) -- the reference computes those with kaolin ON A GPU
    (volsdf_utils.py:172-217), so a CPU run of the reference would not contain them in this form: `value` is the whole step
    (what this port costs on the host), `network_only_rays_per_s` the part a CPU run of the reference's own PyTorch code
    spends in its networks; neither is a like-for-like ratio to quote against the GPU line."""
    sys.path.insert(0, os.path.join(ROOT, "tests"))
    from hold_amd import synthetic as syn
    from oracle import fitting_oracle as fo
    from oracle import geometry_oracle as go
    from oracle import hold_oracle as ho
    from oracle import targets_oracle as to

    # the GPU box exposes 256 hardware threads; torch's intra-op pool stops scaling (and can thrash) far
    # below that on these small per-ray tensors, so the baseline uses the best-measured pool size
    cores = min(threads, os.cpu_count())
    torch.set_num_threads(cores)
    mano = {"right": syn.make_mano_model(True), "left": syn.make_mano_model(False)}
    osc = ho.OracleScene(sc, mano)
    sd = {k: torch.as_tensor(v) for k, v in sd_np.items()}
    frames = [i % sc["n_frames"] for i in range(n_frames)]
    W = 512
    # loss-target meshes of the steady state (what the GPU step has: spawn_cano_mano / meshing_cano): the sealed, once
    # Loop-subdivided canonical MANO (mano_node.py:126-135) and, for the object, a closed mesh of comparable size inside
    # its SDF blob (the object's own canonical mesh comes from marching cubes of the trained SDF; any closed mesh of that
    # size costs the same point-to-mesh work)
    vc = osc.verts_c["right"].reshape(1, 778, 3)
    hv, hf = fo.seal_mano_mesh(vc, torch.as_tensor(np.asarray(mano["right"]["f"], dtype=np.int64)), True)
    hv, hf = to.subdivide_loop(hv[0].numpy(), hf.numpy())
    hv, hf = torch.as_tensor(hv, dtype=torch.float32), torch.as_tensor(hf, dtype=torch.int64)
    ov, of_ = fo.seal_mano_mesh(vc * 0.6, torch.as_tensor(np.asarray(mano["right"]["f"], dtype=np.int64)), True)
    ov, of_ = to.subdivide_loop(ov[0].numpy(), of_.numpy())
    ov, of_ = torch.as_tensor(ov, dtype=torch.float32), torch.as_tensor(of_, dtype=torch.int64)
    bw = ho.barf_weights(4000, 6, 3)
    GEO_SUB = 4  # the off-surface geometry is evaluated on every 4th ray and its time scaled by 4 (~20 instead of ~80 s of host time)
    times, t_net, t_geo = [], [], []
    for rep in range(-1, max(3, repeats)):  # rep -1 = the warm-up (network part only: thread pool, allocator, lazy inits)
        sdg = {k: (v.clone().requires_grad_(True) if v.dtype.is_floating_point else v) for k, v in sd.items()}
        g = torch.Generator().manual_seed(rep + 1)
        pix = torch.randperm(W * W, generator=g)[:128].numpy()
        uv = syn.make_uv(W, W)[pix]
        b = syn.make_batch(sc, frames, uv, W, W)
        inp = {k: torch.from_numpy(v) for k, v in b.items()}
        idx = inp["idx"]
        for nid in sc["entities"]:
            pre = f"nodes.{nid}.params."
            if nid == "object":
                inp["object.global_orient"], inp["object.transl"] = sdg[pre + "global_orient.weight"][idx], sdg[pre + "transl.weight"][idx]
            else:
                inp[f"{nid}.global_orient"], inp[f"{nid}.pose"] = sdg[pre + "global_orient.weight"][idx], sdg[pre + "pose.weight"][idx]
                inp[f"{nid}.transl"] = sdg[pre + "transl.weight"][idx]
                inp[f"{nid}.betas"] = sdg[pre + "betas.weight"][torch.zeros_like(idx)]
        B = len(frames)
        N = B * 128
        rng = {"bg_t": torch.rand(N, 32, generator=g)}
        for n in sc["entities"]:
            rng[n] = {"t_uniform": torch.rand(N, 128, generator=g), "u_final": torch.rand(N, 64, generator=g),
                      "perm": (lambda S: torch.randperm(S))}
        eik = (torch.rand(B, 307, 3, generator=g) - 0.5) * 1.2   # 307 free canonical samples per frame (hold_utils.py:22-55)
        cano = hv[torch.randint(0, hv.shape[0], (B, 307), generator=g)] + 0.01 * torch.randn(B, 307, 3, generator=g)
        t0 = time.time()
        ex = {}
        out = ho.holdnet_forward(osc, sdg, inp, True, rng=rng, current_epoch=0, barf_alpha_iter=4000, extras=ex)
        out["step"], out["epoch"] = 400, 0
        # loss targets (oracle/targets_oracle.py:loss_targets_hand / _object, in float32 and 512-point chunks: the exact
        # point-to-mesh geometry is 1.5e9 point-triangle tests per step, the bulk of the CPU step)
        tg = tg_raw = 0.0  # geometry time as reported (sub-sample scaled to the whole frame) / as spent
        for nid, mv, mf, thr in (("right", hv, hf, 0.01), ("object", ov, of_, 0.05)):
            xc = ex[nid]["x_c"].detach().view(-1, 3)
            tg0 = time.time()
            if rep != 0:  # the exact geometry is deterministic arithmetic without a warm-up effect and 98 % of the step: timed once
                out[f"{nid}.index_off_surface"] = torch.ones(N, dtype=torch.bool)
            else:  # every GEO_SUB-th ray's samples, the time scaled by GEO_SUB (the cost is exactly linear in the points)
                sub = xc.view(N, -1, 3)[::GEO_SUB]
                sdm = go.mesh_sdf(sub.reshape(-1, 3), mv, mf, chunk=512).view(sub.shape[0], -1)
                out[f"{nid}.index_off_surface"] = (sdm.min(dim=1).values > thr).repeat_interleave(GEO_SUB)[:N]
            tg += (time.time() - tg0) * (GEO_SUB if rep == 0 else 1)
            tg_raw += time.time() - tg0
            out[f"{nid}.grad_theta"] = to.grad_theta(sdg, nid, eik, None if nid == "right" else bw)
        tg0 = time.time()
        out["right.pts2mano_sdf_cano"] = (go.mesh_sdf(cano.view(-1, 3), hv, hf, chunk=512).view(B, -1) if rep == 0 else
                                          torch.zeros(B, cano.shape[1]))
        tg += time.time() - tg0
        tg_raw += time.time() - tg0
        xs = cano.reshape(-1, 3)
        out["right.pred_sdf"] = ho.implicit_net(sdg, "nodes.right.implicit_network", xs, torch.zeros(xs.shape[0], 45), 6, None,
                                                zero_cond=True)[:, 0].view(B, -1)
        ld = to.loss_forward({"gt.rgb": torch.from_numpy(b["gt.rgb"]), "gt.mask": torch.from_numpy(b["gt.mask"])}, out)
        ld["loss"].backward()
        if rep >= 0:
            dt_ = time.time() - t0
            if rep == 0:
                t_geo.append(tg)
            t_net.append(dt_ - tg_raw)
    # step = median network part + the geometry part (timed in the first repeat only: see above)
    times = [t + t_geo[0] for t in t_net]
    med = float(np.median(times))
    repeats = len(times)
    # the reference ITSELF cannot run here (a Python reference does not travel to the GPU box): its own training step -- HOLD.training_step
    # with its HOLDNet and Loss, backward, clip, its Adam, 10 frames x 128 rays, no loss-target geometry (steps < 200) -- was timed in
    # the build container (scripts/time_reference_cpu.py) and is QUOTED from the committed record, labelled as what it is
    ref_rec = None
    try:
        ref_rec = json.load(open(os.path.join(ROOT, "profiles", "r06_reference_cpu_step.json")))
        ref_rec["note"] = ("NOT measured on this box: the reference's own training step timed on the build container's CPU cores "
                           "(scripts/time_reference_cpu.py); compare with network_only_rays_per_s, the port's step without the geometry")
    except Exception:
        pass
    return {"value": N / med, "unit": "rays/s", "cores": cores, "kind": "port",
            "reference_timed_in_build_container": ref_rec,
            "repeats": repeats, "step_s": {"median": med, "min": float(min(times)), "max": float(max(times)),
                                           "spread": float((max(times) - min(times)) / med), "all": [round(t, 3) for t in times]},
            "network_only_rays_per_s": N / float(np.median(t_net)),
            "parts_s": {"network_fwd_loss_bwd": [round(t, 3) for t in t_net], "loss_target_geometry": [round(t, 3) for t in t_geo]},
            "like_for_like": False,
            "sample": f"1 warm-up + {repeats} timed training steps of {len(frames)} frames x 128 random pixels = {N} rays -- the reference's step layout "
                      f"(general.yaml:82: 10 frames x 128 = 1 280 rays per step; a bounded sample of it, the cost is linear in frames; "
                      f"--cpu-frames 10 times the whole step: 11.2 rays/s on round 4's box), forward + loss targets (off-surface test of every canonical sample against the "
                      f"{hf.shape[0]}- / {of_.shape[0]}-face loss-target meshes, MANO-canonical SDF, eikonal samples) + the full Loss "
                      f"(rgb, semantics, eikonal, MANO-cano SDF, opacity sparsity) + backward -- the GPU step's terms, without its "
                      f"clip + Adam; median step {med:.2f} s (all: {[round(t, 2) for t in times]}; of which the exact point-to-mesh geometry of the "
                      f"loss targets, kaolin on a GPU in the reference, {float(np.median(t_geo)):.2f} s -- timed once, on every {GEO_SUB}th ray, "
                      f"scaled by {GEO_SUB}; reported apart as parts_s); kind 'port': oracle/hold_oracle.py + "
                      f"oracle/targets_oracle.py, the torch-CPU restatement pinned to the reference by tests/golden -- the reference "
                      f"tree itself is not present on the GPU box; {cores} torch threads of {os.cpu_count()} host hardware threads "
                      f"(torch's intra-op pool stops scaling near 32 on these tensors)"}


# ALGORITHMIC FLOP per ray of SURVEY.md 8(d): linear layers only, 1 MAC = 2 FLOP
F_IMP, F_REND_HAND, F_REND_OBJ, F_BGIMP, F_BGREND = 1_049_088, 532_992, 549_376, 1_065_472, 81_408


def flop_per_ray(node_ids, mean_iters, S, n0, training):
    """sum_n I_n * n0 * F_imp (sampler queries, no grad) + sum_n S * (2 F_imp + F_rend_n) + 32 (F_bgimp + F_bgrend);
    fwd + bwd = sampler term + 3 x the rest (fwd + dX + dW; the reverse sweep is the "2 F_imp")"""
    samp = sum(mean_iters[n] * n0 * F_IMP for n in node_ids)
    rest = sum(S * (2 * F_IMP + (F_REND_OBJ if n == "object" else F_REND_HAND)) for n in node_ids) + 32 * (F_BGIMP + F_BGREND)
    return samp + (3 if training else 1) * rest


def gemm_shapes(prof):
    """aggregate the live launch timings by kernel and (flops per launch) bucket"""
    out = {}
    for e0, e1, fl, name, _nb in prof:
        key = f"{name}:{fl:.3e}"
        a = out.setdefault(key, [0, 0.0, 0.0])
        a[0] += 1
        a[1] += e0.elapsed_time(e1)
        a[2] += fl
    return {k: {"launches": v[0], "ms": v[1], "tflops": v[2] / v[1] / 1e9} for k, v in
            sorted(out.items(), key=lambda kv: -kv[1][1])}


def pmc_traffic(kernel):
    """HBM bytes per launch of `kernel` from the separate rocprofv3 --pmc passes of this same command
    (scripts/pmc.sh -> profiles/<round>_pmc_traffic.json, FETCH_SIZE doubled per the gfx950 calibration)."""
    for rnd in (ROUND,):  # only this round's passes: the kernel families of earlier rounds are other kernels
        f = os.path.join(ROOT, "profiles", f"{rnd}_pmc_traffic.json")
        if os.path.exists(f):
            k = json.load(open(f)).get("kernels", {}).get(kernel)
            if k:
                return k.get("hbm_bytes_per_launch"), os.path.basename(f)
    return None, None


def refine_bench(dev, iters=60):
    """C3's pose-refinement inner loop (optimize_ckpt.py -> fitting/model.py:161-200): iterations/s at B = 10 frames,
    300x300 masks, sealed hand (1 554 faces) + a 5 096-face object."""
    import importlib.util
    spec = importlib.util.spec_from_file_location("bench_fitting", os.path.join(ROOT, "scripts", "bench_fitting.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m.run(iters=iters)


def main():
    args = parse()
    world = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    local = int(os.environ.get("LOCAL_RANK", "0"))
    import torch.distributed as dist

    # stdout carries exactly ONE line, the JSON result of rank 0: native libraries write there too (RCCL prints a version
    # banner to stdout when its communicator comes up), so file descriptor 1 is pointed at stderr for the run and the
    # result goes out through a duplicate of the original descriptor
    sys.stdout.flush()
    json_fd = os.dup(1)
    os.dup2(2, 1)

    force_dist = os.environ.get("HOLD_FORCE_DIST") == "1"  # exercise the RCCL path with a single rank (testing)
    if world > 1 or force_dist:
        os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
        os.environ.setdefault("MASTER_PORT", "29511")
        os.environ.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")
        torch.cuda.set_device(local)
        dist.init_process_group("nccl", rank=rank, world_size=world, device_id=torch.device(f"cuda:{local}"))
    assert world == args.gpus, f"--gpus {args.gpus} but WORLD_SIZE={world}"
    dev = torch.device(f"cuda:{local}")
    torch.cuda.set_device(dev)

    import hold_amd
    from hold_amd import gemm, meshing
    from hold_amd import synthetic as syn
    from hold_amd.hold_net import DEFAULT_SAMPLER
    from hold_amd.loss import Loss
    from hold_amd.optim import FlatAdam, FlatMuon
    from hold_amd.train import render_frame, train_step

    hold_amd.set_precision("f32" if args.fp32_mfma else (args.precision or hold_amd.config.DEFAULT_PRECISION))
    training = args.mode in ("train", "c3")
    W = H = args.res or (1024 if args.mode == "c5" else 512)
    n_frames = max(16, world) if args.mode == "c3" else max(8, world)
    sc = syn.make_scene(n_frames=n_frames, two_hands=args.two_hands)
    sd_np = syn.make_state_dict(sc, barf_iter=3999)
    if args.beta is not None:
        for k in sd_np:
            if k.startswith("nodes.") and k.endswith(".density.beta"):
                sd_np[k] = np.float32(args.beta - 1e-4)  # get_beta() = |beta| + beta_min (1e-4)
    if args.no_compact:
        from hold_amd import field as _fld
        _fld.COMPACT = False
    sampler_opt = dict(DEFAULT_SAMPLER, N_samples=128) if args.mode == "c5" else None
    if args.c2_alt:
        sampler_opt = dict(DEFAULT_SAMPLER, N_samples_eval=64, N_samples=64, N_samples_extra=0)
    net = hold_amd.build_from_scene(sc, sd_np, device=dev, sampler_opt=sampler_opt)
    for node in net.nodes.values():
        node.params.defrost()
        node.implicit_network.embedder_obj.step()
        node.ray_sampler.rng_device = "cuda"  # statistically identical draws without the per-step H2D copy
    net.train(training)
    if not training:
        for node in net.nodes.values():
            node.implicit_network.embedder_obj.eval()
    loss_fn = None
    if training and args.loss == "full":
        # steady-state loss targets (every step after the first canonical-mesh spawn, hold_net.py:154-179): the sealed +
        # subdivided canonical MANO of each hand (spawned at step % 200 == 0) and the object's canonical mesh
        loss_fn = Loss()
        with torch.no_grad():
            obj = net.nodes["object"]
            obj.meshing_cano()  # marching tetrahedra of the object's SDF at the reference's resolution (128^3)
            for nid, node in net.nodes.items():
                if nid != "object":
                    so = node.server(torch.full((1,), sc["scene_scale"], device=dev), node.params.transl.weight[:1],
                                     torch.cat([node.params.global_orient.weight[:1], node.params.pose.weight[:1]], 1),
                                     node.params.betas.weight[:1])
                    node.spawn_cano_mano(so)
    opt = (FlatMuon if args.optimizer == "muon" else FlatAdam)(net, lr=5e-4, clip_norm=0.5) if training else None
    frozen = opt.flat.clone() if (training and not args.no_freeze) else None

    uv = syn.make_uv(W, H)
    if args.mode == "c3":  # the reference's batch: 10 frames x 128 random pixels, a different draw every step
        frames = [(rank * 10 + i) % n_frames for i in range(10)]
        gpix = torch.Generator().manual_seed(1234 + rank)
        batches = []
        for _ in range(4):
            pix = torch.randperm(W * H, generator=gpix)[:args.c3_pixels].numpy()
            bb = syn.make_batch(sc, frames, uv[pix], W, H)
            batches.append({k: torch.from_numpy(v).to(dev) for k, v in bb.items()})
        rays_per_step = 10 * args.c3_pixels
    else:
        split_rays = args.split == "rays" and world > 1
        if split_rays:  # one frame for the whole job; rank r owns rays [r, r + 1) * W * H / world of it
            from hold_amd.parallel import ray_tile, tile_chunks
            lo, hi = ray_tile(W * H, rank, world)
            n_chunks = tile_chunks(W * H, world, args.chunk)  # every rank runs the same number of forwards (collectives inside)
            b = syn.make_batch(sc, [0], uv[lo:hi], W, H)
            for node in net.nodes.values():
                node.ray_sampler.sync_group = True
            if loss_fn is not None:  # the frame's off-surface counts: one scalar all-reduce per node and step (hold_amd.loss)
                loss_fn.sync_group = True
        else:
            b = syn.make_batch(sc, [rank % n_frames], uv, W, H)
        inp = {k: torch.from_numpy(v).to(dev) for k, v in b.items()}
        rays_per_step = inp["uv"].shape[1]
        frame_rays = W * H if split_rays else None  # loss normalisation: the whole frame, so that the tiles' gradients add up
        if not split_rays:
            n_chunks = None
    def step(i):
        if args.mode in ("render", "c5"):
            render_frame(net, inp, args.chunk, n_chunks=n_chunks if args.mode == "render" else None)
            return 0.0
        opt.zero_grad()
        if args.mode == "c3":
            from hold_amd.train import training_step
            bi = batches[i % len(batches)]
            if loss_fn is None:
                loss, _ = train_step(net, bi, args.c3_pixels, step=i + 1, epoch=0)
                lv = loss
            else:
                loss, _, _ = training_step(net, loss_fn, bi, epoch=0, step=i + 1)
                loss.backward()
                lv = loss.detach()
        else:
            lv, _ = train_step(net, inp, args.chunk, step=i + 1, epoch=0, loss_fn=loss_fn, n_total=frame_rays, n_chunks=n_chunks)
        # ray tiles: the all-reduce must SUM the tiles' gradients (FlatAdam averages over ranks: undo it)
        opt.step(grad_mul=float(world) if (args.mode not in ("c3",) and frame_rays is not None) else 1.0)
        if frozen is not None:  # same weights (hence the same SDF, sampler rounds and FLOP per ray) at every step
            opt.flat.copy_(frozen)
        return lv

    for i in range(args.warmup):
        step(i)
    if dist.is_initialized():
        dist.barrier()
    torch.cuda.synchronize()
    if not args.no_profile:
        gemm.PROFILE = []
    from hold_amd import _lib as _L
    for node in net.nodes.values():
        node.ray_sampler.sum_iters = node.ray_sampler.n_calls = 0
    calls0 = _L.CALLS
    from hold_amd import kernels as _K
    ovf0 = _K.h3_overflow_count(dev)  # launches of f16x3 kernels recomputed in f32x6 so far (a host read, outside the timed region)
    if args.sync_debug and rank == 0:
        import collections, traceback, warnings
        sync_sites = collections.Counter()
        def _show(message, category, filename, lineno, file=None, line=None):
            if "synchroniz" not in str(message):
                return
            st = [f for f in traceback.extract_stack()[:-1] if "/hold_amd/" in f.filename or f.filename.endswith("bench.py")]
            sync_sites[" <- ".join(f"{os.path.basename(f.filename)}:{f.lineno}" for f in reversed(st[-4:]))] += 1
        warnings.showwarning = _show
        warnings.simplefilter("always")
        torch.cuda.set_sync_debug_mode("warn")
    tprof = None
    if args.torch_profile and rank == 0:
        from torch.profiler import ProfilerActivity, profile
        tprof = profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA], with_stack=True)
        tprof.__enter__()
    cprof = None
    if args.cprofile and rank == 0:
        import cProfile, functools
        from hold_amd import fitting as _m0, hold_net as _m1, loss as _m2, mano as _m3
        cprof = [cProfile.Profile(), cProfile.Profile()]  # main thread, autograd engine thread

        def _wrap(f):
            @functools.wraps(f)
            def g(*a, **k):
                cprof[1].enable()
                try:
                    return f(*a, **k)
                finally:
                    cprof[1].disable()
            return g
        for m in (_m0, _m1, _m2, _m3):
            for v in list(vars(m).values()):
                if isinstance(v, type) and issubclass(v, torch.autograd.Function) and v is not torch.autograd.Function:
                    v.backward = staticmethod(_wrap(v.backward))
        cprof[0].enable()
    t0 = time.perf_counter()
    rays = 0
    loss = 0.0
    for i in range(args.steps):
        loss = step(args.warmup + i)
        rays += rays_per_step
    torch.cuda.synchronize()
    if args.step_times and rank == 0:  # diagnostic, after the timed region: every further step timed on its own, allocator counters
        keys = ("num_device_alloc", "num_device_free", "num_alloc_retries", "reserved_bytes.all.current", "allocated_bytes.all.peak")
        t_end = time.perf_counter()
        with open(args.step_times, "w") as f:
            for i in range(16):
                m0 = torch.cuda.memory_stats()
                ts = time.perf_counter()
                step(args.warmup + args.steps + i)
                torch.cuda.synchronize()
                m1 = torch.cuda.memory_stats()
                f.write(f"step {i}: {(time.perf_counter() - ts) * 1e3:.1f} ms  " + "  ".join(f"{k} {m0.get(k, 0)} -> {m1.get(k, 0)}" for k in keys) + "\n")
        t0 += time.perf_counter() - t_end  # (not part of the timed region)
    if cprof is not None:
        import io, pstats
        cprof[0].disable()
        with open(args.cprofile, "w") as f:
            for name, p in zip(("main thread (forward, loss, optimiser; backward() = waiting for the engine)", "autograd engine thread (Function.backward bodies)"), cprof):
                for key in ("tottime", "cumulative"):
                    buf = io.StringIO()
                    pstats.Stats(p, stream=buf).sort_stats(key).print_stats(45)
                    f.write(f"# {name}: {args.steps} steps, sorted by {key}\n{buf.getvalue()}\n")
    if args.sync_debug and rank == 0:
        torch.cuda.set_sync_debug_mode("default")
        with open(args.sync_debug, "w") as f:
            f.write(f"# host synchronisation sites over {args.steps} steps of --mode {args.mode} (count, call chain)\n")
            for site, n in sync_sites.most_common():
                f.write(f"{n:6d}  {site}\n")
    if args.op_sites and rank == 0:
        import collections, traceback
        from torch.utils._python_dispatch import TorchDispatchMode
        VIEWS = ("slice", "as_strided", "view", "select", "expand", "permute", "transpose", "reshape", "unsqueeze", "squeeze",
                 "t.", "detach", "alias", "empty", "_unsafe_view", "unbind", "split", "narrow", "size", "stride", "is_", "sym_")
        sites = collections.defaultdict(collections.Counter)

        class _Count(TorchDispatchMode):
            def __torch_dispatch__(self, func, types, a=(), kw=None):
                name = str(func).replace("aten.", "")
                if not name.startswith(VIEWS):
                    st = [f for f in traceback.extract_stack() if "/hold_amd/" in f.filename or f.filename.endswith("bench.py")]
                    st = [f for f in st if "__torch_dispatch__" not in f.name]
                    site = f"{os.path.basename(st[-1].filename)}:{st[-1].lineno} {st[-1].name}" if st else "(autograd engine)"
                    sites[site][name] += 1
                return func(*a, **(kw or {}))

        with _Count():
            step(args.warmup + args.steps)
        torch.cuda.synchronize()
        with open(args.op_sites, "w") as f:
            tot = sum(sum(c.values()) for c in sites.values())
            f.write(f"# non-view torch operators of one --mode {args.mode} step by issuing source line: {tot} in all\n")
            for site, c in sorted(sites.items(), key=lambda kv: -sum(kv[1].values())):
                f.write(f"{sum(c.values()):6d}  {site}  {dict(c.most_common(5))}\n")
    if tprof is not None:
        tprof.__exit__(None, None, None)
        tprof.export_chrome_trace(args.torch_profile + ".trace.json")  # scripts/gap_report.py attributes the device's idle time
        ka = tprof.key_averages()
        with open(args.torch_profile, "w") as f:
            f.write(f"# {args.steps} steps of --mode {args.mode}; sorted by call count\n")
            f.write(ka.table(sort_by="count", row_limit=120, max_name_column_width=70))
            f.write("\n# sorted by device time\n")
            f.write(ka.table(sort_by="cuda_time_total", row_limit=40, max_name_column_width=70))
            f.write("\n# sorted by the host time spent in the operator itself\n")
            f.write(ka.table(sort_by="self_cpu_time_total", row_limit=60, max_name_column_width=70))
            # device-launching aten operators by the hold_amd / bench source line that issued them
            import collections
            sites = collections.defaultdict(lambda: [0, 0.0, collections.Counter()])
            for e in tprof.key_averages(group_by_stack_n=12):
                if not e.key.startswith("aten::") or e.self_device_time_total <= 0:
                    continue
                fr = [x for x in e.stack if "/hold_amd/" in x or "bench.py" in x]
                site = fr[0].split("/")[-1] if fr else "(autograd engine / no python frame)"
                a = sites[site]
                a[0] += e.count; a[1] += e.self_device_time_total; a[2][e.key] += e.count
            f.write("\n# device-launching aten calls by source line: calls, device us, operators\n")
            for site, a in sorted(sites.items(), key=lambda kv: -kv[1][0])[:150]:
                f.write(f"{a[0]:6d} {a[1]:10.0f}  {site}  {dict(a[2].most_common(4))}\n")
    if dist.is_initialized():
        dist.barrier()
    dt = time.perf_counter() - t0
    rank_ms = [dt / args.steps * 1e3]
    if dist.is_initialized():
        # per-rank step times (the first multi-GPU record checks itself: a straggler or a rank that did no work shows here)
        tl = [torch.zeros(1, device=dev, dtype=torch.float64) for _ in range(dist.get_world_size())]
        dist.all_gather(tl, torch.tensor([dt], device=dev, dtype=torch.float64))
        rank_ms = [float(x) / args.steps * 1e3 for x in tl]
        t = torch.tensor([dt], device=dev, dtype=torch.float64)
        dist.all_reduce(t, op=dist.ReduceOp.MAX)
        dt = float(t)
    prof = gemm.PROFILE
    gemm.PROFILE = None

    if rank == 0:
        total_rays = rays * world if not (args.split == "rays" and world > 1 and args.mode != "c3") else args.steps * W * H
        iters = {nid: node.ray_sampler.last_iters for nid, node in net.nodes.items()}
        mean_iters = {nid: node.ray_sampler.sum_iters / max(1, node.ray_sampler.n_calls) for nid, node in net.nodes.items()}
        smp = next(iter(net.nodes.values())).ray_sampler
        S_node = smp.N_samples + 2 + smp.N_samples_extra
        fpr = flop_per_ray(list(net.nodes), mean_iters, S_node, smp.N_samples_eval, training)
        fpr4 = flop_per_ray(list(net.nodes), {n: 4.0 / len(net.nodes) for n in net.nodes}, S_node, smp.N_samples_eval, training)
        x6 = hold_amd.precision() in ("f32x6", "f16x3")
        h3 = hold_amd.precision() == "f16x3"
        # kernel families that run the two-limb fp16 arithmetic in mode f16x3 (3 limb products issued per algorithmic product on
        # v_mfma_f32_32x32x16_f16, same dense peak as bf16); every other split-precision family issues 6 bf16 limb products
        from hold_amd import field as _field
        h3_fams = ({"fused_sdf_kernel", "wgrad_h3_kernel", "rchain_h3_kernel", "rchain_a2_h3_kernel", "rchain_dbwd_h3_kernel", "rchain_bg_h3_kernel", "rgemm_h3_kernel"} |
                   ({"trunk_r6_kernel"} if _field.USE_H3_TRUNK else set())) if h3 else set()
        scene = ("configs[3]-like ARCTIC two-hand (right+left+object+background), " if args.two_hands else
                 "hold_bottle1_itw-like single-hand (right+object+background), ")
        if args.mode == "c3":
            workload = (("configs[2]: the reference's training step -- 10 frames x 128 random pixels = 1 280 rays, " if args.c3_pixels == 128
                         else f"configs[2]-like 10-frame training step at {args.c3_pixels} random pixels per frame = {10 * args.c3_pixels} rays "
                              "(NOT the reference's batch size: --c3-pixels), ") + scene +
                        f"fwd + {'full Loss (loss targets on)' if loss_fn else 'rgb/sem loss'} + bwd incl. pose-table "
                        f"gradients + clip + {'Adam' if args.optimizer == 'adam' else 'FlatMuon'}")
            metric = "rendered rays/sec (fwd+bwd) at the reference's 1 280-ray training batch -- secondary metric (configs[2])"
        elif args.mode == "c5":
            workload = (f"configs[4]: batch render, 1 sequence per GPU, {W}x{H} = {W * H} rays, N_samples = 128 (162 "
                        "samples per fg node), eval forward only, frame stays on the device")
            metric = "rendered rays/sec (forward only, eval mode) at 1024x1024, 128 samples -- secondary metric (configs[4])"
        else:
            workload = ("configs[1]: " + scene + f"1 frame {W}x{H} = {W * H} rays per GPU, " +
                        ("SURVEY 8(d)'s ALTERNATIVE reading of '64+64': 64-sample error-bound hierarchy (N_samples_eval = 64) -> 64 "
                         "importance + 2 samples per fg node (N_samples_extra = 0), 32 bg samples, " if args.c2_alt else
                         "128-sample error-bound hierarchy -> 64 importance + 2 + 32 extra samples per fg node, 32 bg samples, ") +
                        ("fwd + " + ("full reference Loss (eikonal, MANO-cano SDF, opacity-sparsity targets on)" if loss_fn else
                                     "rgb/sem loss") + f" + bwd + grad clip + {'Adam' if args.optimizer == 'adam' else 'FlatMuon'} step" if training else "eval forward only"))
            metric = ("rendered rays/sec (fwd+bwd) at 512x512, 64+64 samples read as N_samples_eval=64 + N_samples=64 -- secondary metric"
                      if (training and args.c2_alt) else "rendered rays/sec (fwd+bwd) at 512x512, 64+64 samples" if training else
                      "rendered rays/sec (forward only, eval mode) -- secondary metric")
        res = {
            "metric": metric, "value": total_rays / dt, "unit": "rays/s", "n_gpus": world, "steps": args.steps,
            "warmup": args.warmup, "ms_per_step": dt / args.steps * 1e3, "higher_is_better": True,
            "scaling": "strong" if (args.split == "rays" and world > 1 and args.mode != "c3") else "weak",
            "vs_baseline": None,
            "dtype": ("f16x3+f32x6 (fp32 results, fp32 accumulation everywhere; the trunk kernels (sampler SDF queries, training forward trunk), the "
                      "three backward sweeps, the single-layer GEMMs of the rendering net and the whole-dW weight gradients split both fp32 "
                      "operands, scaled by exact powers of two -- per matrix for weights, per point / per row / per workgroup for activations and "
                      "loss cotangents -- into two fp16 limbs hi = RN(x), lo = RN(x - hi) and issue hi*hi + hi*lo + lo*hi on "
                      "v_mfma_f32_32x32x16_f16 (3 MFMAs per product, error vs fp64 <= that of f32x6: tests/test_rmlp_gpu.py, test_chain_gpu.py, "
                      "test_gemm_gpu.py; a launch whose scaled operand leaves fp16's range is recomputed in f32x6 by a conditional launch on the "
                      "device: config.f16x3_launches_recomputed_in_f32x6_per_step); gemm_nt, rnarrow, the tile weight gradients and the background's "
                      "sweep are f32x6; --precision f32x6 / --fp32-mfma select the other arithmetics)" if h3 else
                      "f32x6 (fp32 results; every MFMA product = exact 3-limb bf16 split of both fp32 operands, 6 of 9 limb "
                      "products on v_mfma_f32_32x32x16_bf16, fp32 accumulate; --fp32-mfma for true-fp32 operands)"
                      if x6 else "f32"),
            "data": "synthetic",
            "config": {"workload": workload, "chunk_rays": args.chunk if args.mode != "c3" else 10 * args.c3_pixels,
                       "sampler_rounds_last_call": iters, "sampler_rounds_mean_over_timed_calls": mean_iters,
                       "sigma_I": sum(mean_iters.values()),
                       "flop_per_ray": fpr, "flop_per_ray_note": "SURVEY 8(d) algorithmic FLOP (linear layers only) at the "
                       "measured mean sampler rounds of the timed region",
                       "rays_per_s_at_sigmaI_4": total_rays / dt * fpr / fpr4,
                       "algorithmic_tflops_end_to_end": total_rays / dt * fpr / 1e12,
                       "algorithmic_tflops_note": "SURVEY 8(d)'s constants credit every sampler query with lin8's 256 feature rows, "
                       "which the query kernels rightly do not compute (0.918 vs 1.049 MFLOP per point): roofline.end_to_end."
                       "executed_tflops_end_to_end counts the FLOP the MFMA kernels execute",
                       "weights_frozen": frozen is not None,
                       "density_beta": {nid: node.density.beta_host() for nid, node in net.nodes.items()},
                       "sample_compaction": {"enabled": bool(__import__("hold_amd.field", fromlist=["COMPACT"]).COMPACT),
                                             "live_samples_last_call": {nid: getattr(node.field, "last_live", None)
                                                                        for nid, node in net.nodes.items()},
                                             "note": "exact: a sample is dropped behind the sdf only when its Laplace density AND "
                                                     "exp(-|sdf|/beta) are fp32 zeros (hold_amd/csrc/compact.hip); None = every "
                                                     "sample of the last call was live"},
                       "loss_terms": args.loss if training else None,
                       "parallelism": (f"dp{world} (ONE frame, ray tiles per rank, sampler rounds synchronised by a 2-float MAX "
                                       "all-reduce, one RCCL all-reduce (sum) of the flat gradient bucket)"
                                       if (args.split == "rays" and world > 1 and args.mode != "c3") else
                                       f"dp{world} (frames sharded, one RCCL all-reduce of the flat gradient bucket)"),
                       "rccl_ranks": dist.get_world_size() if dist.is_initialized() else 1,
                       "collective_backend": dist.get_backend() if dist.is_initialized() else None,
                       "per_rank_ms_per_step": rank_ms,
                       "loss": float(loss), "precision": hold_amd.precision(),
                       "steps_per_s": args.steps / dt},
        }
        if prof:
            agg, hbm = {}, {}
            for e0, e1, fl, name, nb in prof:
                a = (hbm if name.startswith("hbm:") else agg).setdefault(name, [0.0, 0.0, 0, 0.0])
                a[0] += e0.elapsed_time(e1) * 1e-3
                a[1] += fl
                a[2] += 1
                a[3] += nb
            if args.shape_report:
                json.dump(gemm_shapes(prof), open(args.shape_report, "w"), indent=1)
            split = {"fused_sdf_kernel", "wgrad_kernel", "wgrad_h3_kernel", "chain_kernel", "gemm_nt_kernel", "trunk_r6_kernel", "rchain_kernel",
                     "rchain_bg_kernel", "rchain_a2_kernel", "rchain_dbwd_kernel", "rgemm_kernel", "rnarrow_kernel",
                     "rchain_h3_kernel", "rchain_a2_h3_kernel", "rchain_dbwd_h3_kernel", "rchain_bg_h3_kernel", "rgemm_h3_kernel"} if x6 else set()
            labels = {"gemm_nt_kernel": ("gemm_nt_kernel<x6> (one layer per launch, 3-limb split on v_mfma_f32_32x32x16_bf16)"
                                         if x6 else "gemm_nt_kernel (one layer per launch, v_mfma_f32_32x32x2_f32)"),
                      "trunk_r6_kernel": ("rmlp_h3_kernel<STORE> (forward trunk, 8 layers per launch, register-resident, two fp16 limbs, "
                                          "three products on v_mfma_f32_32x32x16_f16)" if "trunk_r6_kernel" in h3_fams else
                                          "rmlp_kernel<STORE> (forward trunk, 8 layers per launch, register-resident, 3-limb split on "
                                          "v_mfma_f32_32x32x16_bf16)"),
                      "rgemm_kernel": "rgemm_kernel (rendering-net layers, their input gradients, lin8 features: one 256-wide layer "
                                      "per launch, register-resident, 3-limb split on v_mfma_f32_32x32x16_bf16)",
                      "rgemm_h3_kernel": "rgemm_h3_kernel (rendering-net layers, their input gradients, lin8 features: one 256-wide layer "
                                         "per launch, register-resident, two fp16 limbs / three products on v_mfma_f32_32x32x16_f16, every "
                                         "operand row scaled by its own power of two from the producer's row maxima)",
                      "rnarrow_kernel": "rnarrow_kernel (the N <= 64 layers: d sdf / d embedding, the non-feature columns of the colour "
                                        "net's input gradient; A streamed once, ceil(N / 32) output tiles, 3-limb split on "
                                        "v_mfma_f32_32x32x16_bf16)",
                      "rchain_kernel": "rsweep_kernel<DSP> (descending sweep of the normal path, 7 layers per launch, register-resident, "
                                       "side I/O as whole 128-byte lines through LDS, 3-limb split on v_mfma_f32_32x32x16_bf16)",
                      "rchain_bg_kernel": "rsweep_kernel<DSP, skip 172> (the background net's first-order backward sweep, 7 layers per "
                                          "launch, register-resident, 3-limb split on v_mfma_f32_32x32x16_bf16)",
                      "rchain_a2_kernel": "rsweep_kernel<DSP+a2> (first-order backward sweep, 7 layers per launch, register-resident, "
                                          "two side inputs as whole lines through LDS, 3-limb split on v_mfma_f32_32x32x16_bf16)",
                      "rchain_dbwd_kernel": "rsweep_kernel<DBWD> (second-order ascending sweep, 8 layers per launch, register-resident, "
                                            "two side inputs and two results as whole lines through LDS, 3-limb split on "
                                            "v_mfma_f32_32x32x16_bf16)",
                      "rchain_h3_kernel": "rsweep_h3_kernel<DSP> (descending sweep of the normal path, 7 layers per launch, register-resident, "
                                          "two fp16 limbs / three products on v_mfma_f32_32x32x16_f16, per-point operand scales)",
                      "rchain_bg_h3_kernel": "rsweep_h3_kernel<DSP, skip 172> (the background net's first-order backward sweep, two fp16 limbs)",
                      "rchain_a2_h3_kernel": "rsweep_h3_kernel<DSP+a2> (first-order backward sweep, 7 layers per launch, register-resident, "
                                             "two side inputs as whole lines through LDS, two fp16 limbs, per-point operand scales)",
                      "rchain_dbwd_h3_kernel": "rsweep_h3_kernel<DBWD> (second-order ascending sweep, 8 layers per launch, register-resident, "
                                               "two side inputs and two results as whole lines through LDS, two fp16 limbs, per-point "
                                               "operand scales)",
                      "chain_kernel": ("chain_x6_kernel (any sweep not routed to the register-resident kernels: 7-8 trunk layers per launch, "
                                       "LDS-resident, 3-limb split on v_mfma_f32_32x32x16_bf16)" if x6 else
                                       "chain_kernel (7-8 trunk layers per launch, LDS-resident, v_mfma_f32_32x32x2_f32)"),
                      "fused_sdf_kernel": ("rmlp_h3_kernel<HEAD> (sampler SDF queries: register-resident trunk, two fp16 limbs, three "
                                           "products on v_mfma_f32_32x32x16_f16)" if h3 else
                                           "rmlp_kernel<HEAD> (sampler SDF queries: register-resident trunk, 3-limb split on "
                                           "v_mfma_f32_32x32x16_bf16)"
                                           if x6 else "fused_sdf_pipe_kernel (sampler SDF queries, v_mfma_f32_32x32x2_f32)"),
                      "wgrad_h3_kernel": "wgrad_h3_kernel (weight gradients of the 256-wide layers: whole-dW register-resident workgroups, "
                                         "two fp16 limbs / three products on v_mfma_f32_32x32x16_f16, per-workgroup operand scales with "
                                         "exact overflow detection; the 16 / 48-column tail of K = 272 / 304 on the bf16 tile kernel)",
                      "wgrad_kernel": ("wgrad_r6_kernel + wgrad_lds_kernel<x6> (weight gradients: whole-dW register-resident "
                                       "workgroups for the 256x256 layers, LDS tiles otherwise; 3-limb split on v_mfma_f32_32x32x16_bf16)"
                                       if x6 else "wgrad_lds_kernel (weight gradients, v_mfma_f32_32x32x2_f32)")}
            ent = {}
            hbm_step = 0.0
            for name, (t_, fl_, n_, by_) in agg.items():
                tf = fl_ / t_ / 1e12
                is6 = name in split
                nprod = (3.0 if name in h3_fams else 6.0) if is6 else 1.0
                # split-precision kernels are priced on the pipe they run on: 6 bf16 (f16x3 families: 3 fp16) limb products issued
                # per algorithmic product, against the dense bf16 / fp16 MFMA peak; the algorithmic (fp32-equivalent) rate is a
                # named extra
                issued, peak = (nprod * tf, BF16_MFMA_PEAK_TFLOPS) if is6 else (tf, FP32_MFMA_PEAK_TFLOPS)
                # BOTH floors of the family: matrix pipe = issued FLOP / peak; HBM = bytes / 8 TB/s, with the
                # measured bytes (PMC FETCH_SIZE / WRITE_SIZE of separate passes, per launch) when the round's profile has this
                # family and the ALGORITHMIC bytes (operands once, results once) otherwise.  bound = the larger floor.
                pmc_b, pmc_src = pmc_traffic(name)
                alg_b = by_ / n_
                hbm_b = pmc_b if pmc_b else alg_b
                t_launch = t_ / n_
                floor_mfma = (fl_ / n_) * nprod / (peak * 1e12)
                floor_hbm = hbm_b / (HBM_PEAK_GBPS * 1e9)
                bound = "hbm" if floor_hbm > floor_mfma else "mfma"
                hbm_step += hbm_b * n_ / args.steps
                ent[name] = {"bound": bound, "mfma_achieved": issued, "mfma_peak": peak, "mfma_frac": issued / peak,
                             "hbm_achieved_gbps": alg_b / t_launch / 1e9, "hbm_frac": alg_b / t_launch / 1e9 / HBM_PEAK_GBPS,
                             "hbm_frac_measured_bytes": (pmc_b / t_launch / 1e9 / HBM_PEAK_GBPS) if pmc_b else None,
                             "floor_ms": {"mfma": floor_mfma * 1e3, "hbm": floor_hbm * 1e3},
                             "launches": n_, "avg_launch_ms": t_launch * 1e3, "time_share": t_ / dt,
                             "flop_per_launch_avg": fl_ / n_, "algorithmic_bytes_per_launch_avg": alg_b,
                             "traffic": pmc_b, "traffic_source": pmc_src,
                             "arithmetic": ("f16x3" if name in h3_fams else "f32x6") if is6 else "f32",
                             "limb_products_issued_per_product": nprod, "fp32_equivalent_tflops": tf}
                if bound == "hbm":
                    ent[name].update(achieved=alg_b / t_launch / 1e9, peak=HBM_PEAK_GBPS, unit="GB/s",
                                     frac=alg_b / t_launch / 1e9 / HBM_PEAK_GBPS)
                else:
                    ent[name].update(achieved=issued, peak=peak, unit="TFLOP/s", frac=issued / peak)
                if is6:
                    ent[name]["note"] = (f"mfma_achieved = {'fp16' if name in h3_fams else 'bf16'} MFMA FLOP/s issued ({nprod:.0f} limb products per algorithmic fp32 product), "
                                         "mfma_peak = dense bf16 MFMA; fp32_equivalent_tflops = algorithmic FLOP / time; bound = the "
                                         "larger of the two floors (issued FLOP / MFMA peak, HBM bytes / 8 TB/s); achieved / peak / "
                                         "frac are those of the bound")
            # the sampler / compositor stages: scan and search work on <= 640-float per-ray windows held in LDS -- their HBM
            # traffic is the windows in and out; achieved GB/s (algorithmic bytes / live-timed launch) against the HBM roof
            # shows they are nowhere near it (they are latency / LDS-bound at < 2 % of the step), not that they are fast
            for name, (t_, by_, n_, _) in hbm.items():
                ent[name[4:] + "_kernel"] = {"bound": "hbm", "achieved": by_ / t_ / 1e9, "peak": HBM_PEAK_GBPS, "unit": "GB/s",
                                             "frac": by_ / t_ / 1e9 / HBM_PEAK_GBPS, "launches": n_,
                                             "avg_launch_ms": t_ / n_ * 1e3, "time_share": t_ / dt,
                                             "algorithmic_bytes_per_launch_avg": by_ / n_}
            # The top-level object is the dominant kernel TEMPLATE of the step: the sweeps are one kernel template
            # instantiated per mode (rocprof lists rsweep[_h3]_kernel<...> rows), the weight gradients another (whole-dW kernel +
            # its tile / reduction helpers stay separate families here).  A template's numbers are those of its families taken
            # together: time-weighted, i.e. total FLOP, total bytes, total time, per average launch.
            template_of = {"rchain_kernel": "rsweep_kernel", "rchain_a2_kernel": "rsweep_kernel", "rchain_dbwd_kernel": "rsweep_kernel",
                           "rchain_bg_kernel": "rsweep_kernel", "rchain_h3_kernel": "rsweep_h3_kernel",
                           "rchain_a2_h3_kernel": "rsweep_h3_kernel", "rchain_dbwd_h3_kernel": "rsweep_h3_kernel",
                           "rchain_bg_h3_kernel": "rsweep_h3_kernel"}
            tmpl = {}
            for name in agg:
                tmpl.setdefault(template_of.get(name, name), []).append(name)
            dom_t = max(tmpl, key=lambda t: sum(ent[k]["time_share"] for k in tmpl[t]))
            fams = tmpl[dom_t]
            if len(fams) == 1:
                dom = fams[0]
                d = ent[dom]
            else:
                dom = dom_t
                n_ = sum(agg[k][2] for k in fams)
                t_ = sum(agg[k][0] for k in fams)
                fl_iss = sum(agg[k][1] * ent[k]["limb_products_issued_per_product"] for k in fams)
                fl_ = sum(agg[k][1] for k in fams)
                alg_b = sum(agg[k][3] for k in fams)
                have_pmc = all(ent[k]["traffic"] for k in fams)
                pmc_b = sum(ent[k]["traffic"] * agg[k][2] for k in fams) if have_pmc else None
                peak = ent[fams[0]]["mfma_peak"]
                floor_mfma, floor_hbm = fl_iss / (peak * 1e12) / n_, (pmc_b if pmc_b else alg_b) / (HBM_PEAK_GBPS * 1e9) / n_
                d = {"bound": "hbm" if floor_hbm > floor_mfma else "mfma", "mfma_achieved": fl_iss / t_ / 1e12, "mfma_peak": peak,
                     "mfma_frac": fl_iss / t_ / 1e12 / peak, "hbm_frac": alg_b / t_ / 1e9 / HBM_PEAK_GBPS,
                     "hbm_frac_measured_bytes": (pmc_b / t_ / 1e9 / HBM_PEAK_GBPS) if pmc_b else None,
                     "floor_ms": {"mfma": floor_mfma * 1e3, "hbm": floor_hbm * 1e3}, "launches": n_, "avg_launch_ms": t_ / n_ * 1e3,
                     "time_share": t_ / dt, "flop_per_launch_avg": fl_ / n_, "algorithmic_bytes_per_launch_avg": alg_b / n_,
                     "traffic": (pmc_b / n_) if pmc_b else None, "traffic_source": ent[fams[0]]["traffic_source"],
                     "arithmetic": ent[fams[0]]["arithmetic"], "fp32_equivalent_tflops": fl_ / t_ / 1e12,
                     "note": "one kernel template, its instantiations taken together (time-weighted): " + ", ".join(
                         f"{k} {ent[k]['time_share'] * 100:.1f} %" for k in sorted(fams, key=lambda k: -ent[k]["time_share"])) +
                         "; each is listed on its own under kernels"}
                if d["bound"] == "hbm":
                    d.update(achieved=alg_b / t_ / 1e9, peak=HBM_PEAK_GBPS, unit="GB/s", frac=alg_b / t_ / 1e9 / HBM_PEAK_GBPS)
                else:
                    d.update(achieved=d["mfma_achieved"], peak=peak, unit="TFLOP/s", frac=d["mfma_frac"])
                labels[dom] = (f"{dom} (csrc/rchain{'_h3' if 'h3' in dom else ''}.hip: the register-resident backward sweeps -- DSP, "
                               "DSP+a2, DBWD instantiations of one template)")
            res["roofline"] = {"bound": d["bound"], "achieved": d["achieved"], "peak": d["peak"], "unit": d["unit"],
                               "frac": d["frac"], "traffic": d["traffic"],
                               "mfma_frac": d["mfma_frac"], "hbm_frac": d["hbm_frac"],
                               "hbm_frac_measured_bytes": d["hbm_frac_measured_bytes"], "floor_ms": d["floor_ms"],
                               "kernel": labels.get(dom, dom), "launches": d["launches"],
                               "avg_launch_ms": d["avg_launch_ms"], "time_share": d["time_share"],
                               "flop_per_launch_avg": d["flop_per_launch_avg"],
                               "algorithmic_bytes_per_launch_avg": d["algorithmic_bytes_per_launch_avg"],
                               "arithmetic": d["arithmetic"],
                               "fp32_equivalent_tflops": d["fp32_equivalent_tflops"],
                               "traffic_note": (f"HBM bytes/launch of this kernel from separate --pmc passes (profiles/{d['traffic_source']})"
                                                if d["traffic"] else "no PMC pass of this kernel family in profiles/ yet"),
                               "kernels": ent}
            if "note" in d:
                res["roofline"]["note"] = d["note"]
            mf = sum(v[1] for v in agg.values())
            mf6 = sum(((3.0 if k in h3_fams else 6.0) if k in split else 1.0) * v[1] for k, v in agg.items())
            res["roofline"]["end_to_end"] = {"mfma_tflops_fp32_equivalent": mf / dt / 1e12,
                                             "executed_tflops_end_to_end": mf / dt / 1e12,
                                             "mfma_tflops_issued": mf6 / dt / 1e12,
                                             "frac_of_bf16_mfma_peak_issued": (mf6 / dt / 1e12 / BF16_MFMA_PEAK_TFLOPS) if x6 else None,
                                             "frac_of_fp32_mfma_peak": None if x6 else mf / dt / 1e12 / FP32_MFMA_PEAK_TFLOPS,
                                             "time_in_mfma_kernels": sum(v[0] for v in agg.values()) / dt,
                                             # HBM side of the whole step: bytes of the MFMA families (PMC per launch where
                                             # profiled, algorithmic otherwise) x launches; floors of the step on both roofs
                                             "hbm_bytes_per_step": hbm_step,
                                             "hbm_tb_s": hbm_step / (dt / args.steps) / 1e12,
                                             "hbm_frac_of_8tbs": hbm_step / (dt / args.steps) / (HBM_PEAK_GBPS * 1e9),
                                             "step_floor_s": {"hbm": hbm_step / (HBM_PEAK_GBPS * 1e9),
                                                              "mfma": mf6 / args.steps / ((BF16_MFMA_PEAK_TFLOPS if x6 else FP32_MFMA_PEAK_TFLOPS) * 1e12)}}
        res["config"]["c_abi_calls_per_step"] = (_L.CALLS - calls0) / args.steps
        res["config"]["f16x3_launches_recomputed_in_f32x6_per_step"] = (_K.h3_overflow_count(dev) - ovf0) / args.steps
        res["config"]["f16x3_fallback_note"] = ("overflow guard of the f16x3 kernels (trunk, sampler queries, backward sweeps): a launch in which a "
                                                "scaled operand left fp16's range is recomputed by a conditional f32x6 launch on the device")
        if args.mode == "c3" and not args.no_refine:
            try:
                res["config"]["pose_refine"] = refine_bench(dev)
            except Exception as e:  # the refinement leg is reported beside the step rate, never instead of it
                res["config"]["pose_refine"] = {"error": repr(e)}
        if not args.no_cpu_baseline and world == 1 and args.mode == "train" and not args.two_hands:
            res["cpu_baseline"] = cpu_baseline(sc, sd_np, args.cpu_threads, n_frames=args.cpu_frames)
        os.write(json_fd, (json.dumps(res) + "\n").encode())
    if dist.is_initialized():
        dist.destroy_process_group()


if __name__ == "__main__":
    main()
