#!/usr/bin/env python
"""Throughput of the ImmunoStruct train step on MI355X (BASELINE.json metric).

    python bench.py --gpus N --steps K --warmup W [--workload iedb|paired|stress]

A "step" = one pass of the hot path over one batch of synthetic peptide-MHC residue graphs already resident in HBM.

``iedb`` (default; BASELINE config 2 / 3): HybridModelv2 forward (6 EGNN layers -> node attention -> mean-pool, sequence
    VAE, property MLP, fusion head) + regression loss + backward + Adam -- the inner loop of ``procedures/train.py:18-29``
    with ``--full-sequence --sequence-loss``, B = 128 graphs of 190 padded nodes per GPU.
``paired`` (config 4): HybridModelv2_Comparative, ``--use-wt-for-downstream``, BCE + 0.01 x paired contrastive loss,
    AdamW -- ``procedures/train.py:84-123`` / ``utils/contrastive.py:37-83`` -- B = 128 (cancer, wild-type) pairs =
    256 graphs per GPU and step.
``stress`` (config 5, one GPU's slice): the 6-layer EGNN stack alone, forward + backward (all weight gradients), on
    random residue graphs of ~200 nodes (clipped N(200, 15), padded to the slice's maximum), 8 edge features,
    average in-degree 8, 64 node channels; B = 256 graphs per GPU and step.

N > 1: one process per GPU (``torch.distributed.run``, or this script launches its own ranks when started as plain
``python bench.py --gpus N``), graphs sharded over ranks (weak scaling), one RCCL all-reduce of the flat gradient per
step.  Rank 0 prints ONE JSON line with the contract fields plus
  "roofline"     -- the dominant HIP kernel (fused EGNN layer backward): algorithmic FLOP / launch divided by its mean
                    launch duration (HIP events on the launching stream), against the fp32 MFMA peak; the HBM view of the
                    same launches, the forward layer kernel and (when it still runs) the pure gather kernel next to it.
  "cpu_baseline" -- the CPU oracle (a port of the reference's un-fused PyTorch path) timed on this box's host cores on a
                    bounded sample of the same workload (N = 1, rank 0 only).
"""
from __future__ import annotations

import argparse
import gc
import json
import os
import sys
import time

import numpy as np
import torch

ROOT = os.path.dirname(os.path.abspath(__file__))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

from immunostruct_amd import distributed as D  # noqa: E402
from immunostruct_amd import functional as HF  # noqa: E402
from immunostruct_amd import optim  # noqa: E402
from immunostruct_amd import synthetic  # noqa: E402
from immunostruct_amd.graph import PackedGraphBatch  # noqa: E402
from immunostruct_amd.models import model_map  # noqa: E402
from immunostruct_amd.utils import Losses  # noqa: E402

VAE_IN = synthetic.SEQ_LEN * synthetic.SEQ_ALPHABET
PEAK_FP32_MFMA_TFLOPS = 157.3   # MI355X_MICROARCH.md: Peak FP32 (matrix)
PEAK_HBM_GBS = 8000.0           # MI355X_MICROARCH.md: HBM3E peak BW (spec)
H = 64
# where the captured step's dropout masks / reparameterisation noise come from (engine.CapturedTrainStep step_random):
# "device" = one launch of the library's generator inside the step, as the device-resident training loops of ``procedures`` run it
# (None would be torch's generator inside the step: two generator-state fills in front of every replay)
STEP_RANDOM = "device"
TRAFFIC_FILE = os.path.join("profiles", "r06_pmc_traffic.json")   # PMC-measured HBM bytes per launch (profiles/README.md)


def layer_algorithmic(n_nodes, n_edges, din, fe):
    """Algorithmic bytes / FLOP of one EGNN layer launch.

    bytes: SURVEY's per-layer figure (it already holds the node rows: self rows for the node MLP / coordinate update and
    the writes).  FLOP: the dense work the launch performs -- edge half: the per-edge layers that remain after hoisting the
    first edge-MLP layer to node level (forward 2 x 64x64 + 64; backward 2 data-gradient + 2 weight-gradient 64x64
    products); node half (in the same launch since round 2): forward node MLP (Din+64 -> 64 -> 64) + the next 64 -> 128
    pre-projection, backward their three data-gradient products.  Returns (bytes_fwd, bytes_bwd, flop_fwd, flop_bwd,
    edge-only flop_fwd, edge-only flop_bwd).
    """
    bytes_fwd = n_edges * (2 * din * 4 + 24 + fe * 4 + 4) + (n_nodes + 1) * 4 + n_nodes * (din * 4 + 12) + n_nodes * (H * 4 + 12)
    bytes_bwd = n_edges * (2 * din * 4 + 24 + fe * 4 + 4) + n_nodes * H * 4 + 2 * n_nodes * (din + 3) * 4
    edge_fwd = 2.0 * n_edges * (H * H + H * H + H)
    edge_bwd = 2.0 * n_edges * (4 * H * H + 2 * H)
    node = 2.0 * n_nodes * ((din + H) * H + H * H + H * 2 * H)
    return bytes_fwd, bytes_bwd, edge_fwd + node, edge_bwd + node, edge_fwd, edge_bwd


def measured_copy_ceiling(dev, gib=1.0):
    """the copy-bandwidth ceiling of THIS device (HBM fractions "also against a measured hipMemcpy /
    triad ceiling"): csrc/abi_misc.hip ``is_debug_stream_copy`` (16-byte non-temporal loads / stores) over ``gib`` GiB each way --
    far beyond the 256 MB of L2 + MALL -- timed with HIP events, best of several grids; torch's own device-to-device copy
    (hipMemcpyAsync's kernel) beside it.  Bytes counted = read + written."""
    from immunostruct_amd import _lib
    lib = _lib.load()
    n16 = int(gib * (1 << 30)) // 16
    src = torch.empty(n16 * 4, dtype=torch.float32, device=dev).normal_()
    dst = torch.empty_like(src)
    st = _lib.stream_ptr()

    def timed(fn, reps=5):
        fn()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        best = None
        for _ in range(reps):
            a.record(); fn(); b.record(); b.synchronize()
            ms = a.elapsed_time(b)
            best = ms if best is None else min(best, ms)
        return 32.0 * n16 / (best * 1e-3) / 1e9
    by_grid = {}
    for grid in (2048, 4096, 8192, 16384):
        by_grid[str(grid)] = round(timed(lambda: _lib.check(lib.is_debug_stream_copy(_lib.ptr(src), _lib.ptr(dst), n16, grid, st),
                                                            "is_debug_stream_copy")), 1)
    memcpy = round(timed(lambda: dst.copy_(src)), 1)
    ok = bool(torch.equal(src[:4096], dst[:4096]) and torch.equal(src[-4096:], dst[-4096:]))
    del src, dst
    return dict(value=max(max(by_grid.values()), memcpy), unit="GB/s", stream_copy_by_grid=by_grid, torch_copy=memcpy, copied_ok=ok,
                bytes_each_way=n16 * 16, what="device-to-device copy, read + written bytes / best-of-5 duration (HIP events)")


def attach_measured_peak(roof, ceiling):
    """every HBM-view fraction of the roofline object also against the measured copy ceiling"""
    if roof is None or ceiling is None:
        return
    peak = ceiling["value"]
    hv = roof["hbm_view"]
    hv["measured_peak"], hv["frac_of_measured"] = peak, round(hv["achieved"] / peak, 4)
    hv["measured_peak_detail"] = ceiling
    if roof.get("traffic"):
        us = roof["mean_launch_us"]
        hv["traffic_gbs"] = round(roof["traffic"] / (us * 1e-6) / 1e9, 1)
        hv["traffic_frac_of_measured"] = round(hv["traffic_gbs"] / peak, 4)
    fk = roof["forward_kernel"]
    fk["frac_hbm_of_measured"] = round(fk["hbm_gbs"] / peak, 4)
    if "gather_kernel" in roof:
        gk = roof["gather_kernel"]
        gk["measured_peak"], gk["frac_of_measured"] = peak, round(gk["achieved"] / peak, 4)


def kernel_sources_sha256():
    """digest of the sources the layer kernels are built from: a PMC traffic figure measured for other sources is stale"""
    import hashlib
    h = hashlib.sha256()
    for name in ("egnn_layer_fwd.hip", "egnn_layer_bwd.hip", "egnn_layer_bwd8.hip", "common.h", "node16.h"):
        with open(os.path.join(ROOT, "immunostruct_amd", "csrc", name), "rb") as f:
            h.update(f.read())
    return h.hexdigest()


def measured_traffic(traffic_key):
    """(bytes per egnn_layer_bwd launch | None, where it comes from / why it is missing)"""
    tpath = os.path.join(ROOT, TRAFFIC_FILE)
    if traffic_key is None:
        return None, "no PMC measurement for this batch size / density"
    if not os.path.isfile(tpath):
        return None, f"{TRAFFIC_FILE} not found"
    rec = json.load(open(tpath))
    want, have = kernel_sources_sha256(), rec.get("kernel_sources_sha256")
    if have != want:
        return None, (f"{TRAFFIC_FILE} was measured for other kernel sources (sha256 {str(have)[:12]}..., this tree {want[:12]}...): "
                      f"re-run tools/pmc_traffic.sh")
    ent = rec.get(traffic_key, {}).get("egnn_layer_bwd_kernel")
    if not ent:
        return None, f"{TRAFFIC_FILE} holds no {traffic_key} entry"
    return ent.get("bytes"), f"{TRAFFIC_FILE} ({rec.get('commit', '?')}): separate rocprofv3 --pmc passes of this workload, same kernel sources"


def _paired_bwd_in_use(n_nodes, n_edges, fe):
    """whether the backward layer launches of this batch run as the paired 512-thread kernel (functional.use_paired_bwd's rule)"""
    return bool(HF.use_paired_bwd(int(n_nodes), fe))


def roofline_from_timers(timers, n_nodes, n_edges, dins, fe, traffic_key, insitu=None, paired_bwd=False):
    """``dins``: input width of the layers whose launches run the FULL pass (coordinate branch included).
    ``insitu``: {"bwd": {"slot": [us ...], "span": [...]}, "fwd": ..., "gather": ...} from the workgroup clocks of the REPLAYED
    step (functional.LaunchClock.durations) -- the primary timing of every entry is the ``slot`` time (end of the previous layer
    launch -> end of this one: dispatch gap and ramp included, what a kernel trace reports for back-to-back launches);
    ``timers`` (HIP events around eager launches) are reported as the secondary ``eager_us`` figures.  Without ``insitu``
    (``--eager`` / ``--no-kernel-timers`` runs) the HIP events are used."""
    ev = {k: timers[k][1] * 1e3 for k in ("egnn_layer_bwd", "egnn_layer_fwd", "gather_segment_sum") if k in timers}
    src = {}
    for key, name in (("bwd", "egnn_layer_bwd"), ("fwd", "egnn_layer_fwd"), ("gather", "gather_segment_sum")):
        if insitu and insitu.get(key) and insitu[key]["slot"]:
            src[key] = (float(np.mean(insitu[key]["slot"])), len(insitu[key]["slot"]), "insitu")
        elif name in ev:
            src[key] = (ev[name], timers[name][0], "events")
    if "bwd" not in src or "fwd" not in src:
        return None
    per = [layer_algorithmic(n_nodes, n_edges, din, fe) for din in dins]
    b_fwd, b_bwd = np.mean([p[0] for p in per]), np.mean([p[1] for p in per])
    f_fwd, f_bwd = np.mean([p[2] for p in per]), np.mean([p[3] for p in per])
    e_fwd, e_bwd = np.mean([p[4] for p in per]), np.mean([p[5] for p in per])
    (us_b, n_b, how), (us_f, n_f, _) = src["bwd"], src["fwd"]
    tf_b, tf_f = f_bwd / (us_b * 1e-6) / 1e12, f_fwd / (us_f * 1e-6) / 1e12
    traffic, traffic_src = measured_traffic(traffic_key)
    method = ("workgroup clocks inside the launches of the REPLAYED step (every workgroup stores the device wall clock at its start "
              "and end; csrc/common.h wg_clock_*): a launch is charged from the last workgroup end of the previous layer launch to "
              "its own last workgroup end (its slot on the step's critical chain, dispatch gap and ramp included; `insitu_us.*.span` "
              "= first start to last end of the launch alone) -- the same captured graph whose throughput is `value`, co-running "
              "branches included" if how == "insitu" else
              "HIP events on the launching stream around eager launches")
    sec = lambda name: round(ev[name], 2) if (how == "insitu" and name in ev) else None
    roof = dict(kernel="egnn_layer_bwd8_kernel (paired: one 512-thread workgroup per CU)" if paired_bwd else "egnn_layer_bwd_kernel", bound="mfma", achieved=round(tf_b, 2), peak=PEAK_FP32_MFMA_TFLOPS, unit="TFLOP/s",
                frac=round(tf_b / PEAK_FP32_MFMA_TFLOPS, 4), traffic=traffic, traffic_source=traffic_src, launches=n_b,
                mean_launch_us=round(us_b, 2), timing=method, eager_us=sec("egnn_layer_bwd"),
                algorithmic_flop_per_launch=f_bwd, algorithmic_bytes_per_launch=b_bwd,
                edge_half_only=dict(algorithmic_flop_per_launch=e_bwd, tflops=round(e_bwd / (us_b * 1e-6) / 1e12, 2),
                                    frac=round(e_bwd / (us_b * 1e-6) / 1e12 / PEAK_FP32_MFMA_TFLOPS, 4),
                                    note="FLOP of the per-edge products only over the whole launch's duration (round 1's accounting, "
                                         "when the node data path and the source gather were their own launches)"),
                hbm_view=dict(achieved=round(b_bwd / (us_b * 1e-6) / 1e9, 1), peak=PEAK_HBM_GBS, unit="GB/s",
                              frac=round(b_bwd / (us_b * 1e-6) / 1e9 / PEAK_HBM_GBS, 4)),
                forward_kernel=dict(kernel="egnn_layer_fwd_kernel", mean_launch_us=round(us_f, 2), launches=n_f,
                                    eager_us=sec("egnn_layer_fwd"), tflops=round(tf_f, 2), frac_mfma=round(tf_f / PEAK_FP32_MFMA_TFLOPS, 4),
                                    edge_half_only_frac_mfma=round(e_fwd / (us_f * 1e-6) / 1e12 / PEAK_FP32_MFMA_TFLOPS, 4),
                                    hbm_gbs=round(b_fwd / (us_f * 1e-6) / 1e9, 1),
                                    frac_hbm=round(b_fwd / (us_f * 1e-6) / 1e9 / PEAK_HBM_GBS, 4)))
    if "gather" in src:
        us_g, n_g, _ = src["gather"]
        gbytes = n_edges * (H * 4 + 12 + 4) + n_nodes * (H * 4 + 12 + 4)
        roof["gather_kernel"] = dict(kernel="gather_segment_sum_kernel", bound="hbm", mean_launch_us=round(us_g, 2),
                                     launches=n_g, eager_us=sec("gather_segment_sum"), achieved=round(gbytes / (us_g * 1e-6) / 1e9, 1),
                                     unit="GB/s", frac=round(gbytes / (us_g * 1e-6) / 1e9 / PEAK_HBM_GBS, 4),
                                     note="one launch per step (layer 0); the other layers' source gathers run inside "
                                          "egnn_layer_bwd_kernel")
    return roof


def timed_cpu(step, units_per_step, budget_s, what, loader_step=None):
    """the CPU oracle's ``step`` on this box's host cores as SURVEY.md section 8(d)(ii) asks: all cores AND one thread, on a
    pre-batched input AND (``loader_step``: the same step behind the oracle's per-step batch construction -- ``dgl.batch``
    restated + one-hot expansion -- the reference's DataLoader work, ``data/utils.py:160-176``) batch-construction-inclusive.
    These small un-fused ops do not scale to hundreds of threads, so a 16-thread sample is taken too; the headline ``value`` is
    the best pre-batched sample, every sample is in the object.  Bounded to ~``budget_s`` seconds in total."""
    all_threads = torch.get_num_threads()

    def sample(fn, threads, seconds, max_steps):
        torch.set_num_threads(threads)
        fn()  # warm-up
        t0, n = time.perf_counter(), 0
        while True:
            fn()
            n += 1
            if time.perf_counter() - t0 > seconds or n >= max_steps:
                break
        dt = time.perf_counter() - t0
        return dict(value=round(units_per_step * n / dt, 2), unit="graphs/s", cores=threads, steps=n, seconds=round(dt, 1))

    share = budget_s / (4.5 if loader_step is not None else 3.5)
    out = {"all_cores": sample(step, all_threads, share, 40)}
    if all_threads > 16:
        out["threads_16"] = sample(step, 16, share, 40)
    out["one_thread"] = sample(step, 1, share / 2, 3)
    best_key = max((k for k in out if k != "one_thread"), key=lambda k: out[k]["value"])
    if loader_step is not None:
        out["with_batch_construction"] = sample(loader_step, out[best_key]["cores"], share, 40)
    torch.set_num_threads(all_threads)
    best = out[best_key]
    res = dict(value=best["value"], unit="graphs/s", cores=best["cores"], kind="port",
               sample=f"{best['steps']} steps of {what}, {best['cores']} torch threads of {all_threads} available, {best['seconds']} s "
                      f"(headline = best pre-batched sample; all_cores / threads_16 / one_thread / with_batch_construction beside it)",
               host_threads_available=all_threads)
    res.update(out)
    return res


# ---------------------------------------------------------------------------------------------------------------------
# workloads: each offers  step(i) / eager_step(i) / graphs_per_step / describe() / roofline(timers) / cpu_baseline() /
# extra_config() / eager_timers_setup()
# ---------------------------------------------------------------------------------------------------------------------
def device_batch(raw, dev, y_key):
    g = PackedGraphBatch.from_raw(raw, device=dev)
    return dict(g=g, seq=torch.from_numpy(raw.one_hot_sequence()).to(dev), prop=torch.from_numpy(raw.prop).to(dev),
                y=torch.from_numpy(getattr(raw, y_key)).to(dev), raw=raw)


class TrainStepWorkload:
    """shared by ``iedb`` and ``paired``: model + loss + optimizer behind the captured HIP-graph step"""

    def _finish(self, args, world, template, edge_capacity):
        self.reducer = D.FlatGradReducer(self.model.parameters(), world=world, always_pack=args.force_pack)
        self.captured = None
        if not args.eager:
            from immunostruct_amd.engine import CapturedTrainStep
            self.captured = CapturedTrainStep(self.model, self.opt, self.reducer, self.forward_loss, template,
                                              edge_capacity=edge_capacity, step_random=STEP_RANDOM)

    def step(self, i):
        if self.captured is None:
            return self.eager_step(i)
        return self.captured(*self.batch(i))

    def eager_step(self, i):
        self.reducer.zero()
        loss = self.forward_loss(self.model, *self.batch(i))
        loss.backward()
        self.reducer.all_reduce_mean()
        self.opt.step()
        return loss.detach()

    def eager_timers_setup(self):
        """per-kernel timers run on an eager, single-stream re-run: the sequence branch on the SAME stream (a kernel's
        duration is then its own, not the co-run slow-down by the forked branch), gradients packed from the live tensors"""
        from immunostruct_amd.models import _core as model_core
        saved = model_core.OVERLAP_BRANCHES
        model_core.OVERLAP_BRANCHES = False
        for bucket in self.reducer.buckets:
            bucket["sources"] = None

        def restore():
            model_core.OVERLAP_BRANCHES = saved
        return restore

    def extra_config(self):
        c, r = self.captured, self.reducer
        if c is None or not r.packing:
            return dict(launch="eager" if c is None else "hipGraph replay", grad_allreduce=None)
        # everything a multi-GPU line needs to explain its own efficiency: the form the engine kept and the step time of every
        # form it timed at construction (serial; two-stage per number of reserved CUs), the standalone all-reduce time of every
        # bucket (all ranks call this: it holds collectives), and the RCCL channel bound in effect
        return dict(launch="hipGraph replay",
                    grad_allreduce=dict(form=({"graph": "one graph: serial, collectives captured",
                                               "graph2": "one graph: two-stage backward, bucket 0 overlapped, collectives captured"}[c.one_graph]
                                              if c.one_graph else
                                              ("two-stage backward, bucket 0 overlapped" if c.two_stage else "serial")),
                                        one_graph_error=c.one_graph_error,
                                        reserved_cus=c.reserved if (c.two_stage and not c.one_graph) else None,
                                        buckets=[int(b["flat"].numel()) for b in r.buckets], tuned_ms=c.dp_times,
                                        standalone_allreduce=D.time_all_reduce(r),
                                        nccl_max_nchannels=os.environ.get("NCCL_MAX_NCHANNELS"),
                                        nccl_min_nchannels=os.environ.get("NCCL_MIN_NCHANNELS")))


class IedbWorkload(TrainStepWorkload):
    name = "iedb"

    def __init__(self, args, dev, rank, world):
        self.args = args
        torch.manual_seed(1)
        self.model = model_map[args.model](vae_input_dim=VAE_IN, device=dev).to(dev)
        D.broadcast_parameters(self.model)
        self.model.train()
        # stage "pretrain": regression on the normalised foreignness, Adam lr 1e-3 (train_IEDB_wFT.py:74-88); stage "finetune":
        # BCE on immunogenicity, Adam lr 1e-4, weight decay 1e-6 (train_IEDB_wFT.py:97-113) -- config 2's second stage
        self.finetune = args.stage == "finetune"
        if self.finetune:
            self.opt = optim.Adam(self.model.parameters(), lr=1e-4, weight_decay=1e-6)      # csrc/optimizer.hip
        else:
            self.opt = optim.Adam(self.model.parameters(), lr=1e-3)
        self.losses = Losses(VAE_IN, {0: 81.0, 1: 19.0}, sequence=True)
        self.pool = [device_batch(synthetic.make_batch(args.batch, seed=1000 * (rank + 1) + i, deg_extra=args.deg_extra,
                                                       symmetric=args.symmetric_edges), dev,
                                  "y_bin" if self.finetune else "y_reg") for i in range(4)]
        self.graphs_per_step = args.batch
        self.n_nodes = self.pool[0]["raw"].num_nodes
        self.n_edges = float(np.mean([b["raw"].num_edges for b in self.pool]))
        self._finish(args, world, self.batch(0), max(b["raw"].num_edges for b in self.pool))

    def forward_loss(self, m, g, seq, prop, y):
        recon, mu, logvar, final = m(g, seq, prop)
        if self.finetune:
            return self.losses.BCE_loss(recon, seq, mu, logvar, final, y)
        return self.losses.regression_loss(recon, seq, mu, logvar, final, y)
    forward_loss.fused_loss = True      # (utils.Losses only: engine.CapturedTrainStep may let the head join the sequence branch early)

    def batch(self, i):
        b = self.pool[i % len(self.pool)]
        return b["g"], b["seq"], b["prop"], b["y"]

    def describe(self):
        a = self.args
        if self.finetune:
            return (f"IEDB finetune step (BASELINE config 2, second stage): {a.model}, full-sequence + sequence-loss, BCE loss "
                    f"(pos_weight 81/19), Adam lr 1e-4 weight decay 1e-6; B={a.batch} graphs/GPU x 190 padded nodes, "
                    f"E~{int(self.n_edges)} edges/batch (deg_extra={a.deg_extra}), Fe=1")
        return (f"IEDB pretrain step (BASELINE config 2): {a.model}, full-sequence + sequence-loss, regression loss, Adam; "
                f"B={a.batch} graphs/GPU x 190 padded nodes, E~{int(self.n_edges)} edges/batch (deg_extra={a.deg_extra}"
                f"{', every edge in both directions' if a.symmetric_edges else ''}), Fe=1")

    def roofline(self, timers, insitu=None):
        # the timed launches are the five full ones per step (layer 0: Din = 20, layers 1-4: Din = 64); the last layer's
        # launch skips the coordinate MLP (its output is unused by the model) and is timed under its own name
        key = "iedb_B128_deg2" if (self.args.batch == 128 and self.args.deg_extra == 2 and not self.args.symmetric_edges) else None
        return roofline_from_timers(timers, self.n_nodes, self.n_edges, (20, 64, 64, 64, 64), 1, key, insitu,
                                    paired_bwd=_paired_bwd_in_use(self.n_nodes, self.n_edges, 1))

    def cpu_baseline(self, budget_s=24.0):
        from oracle import functional_ref as FR
        from oracle import graph_ref
        a = self.args
        raw = synthetic.make_batch(a.batch, seed=1, deg_extra=a.deg_extra, symmetric=a.symmetric_edges)
        shapes = {k: tuple(v.shape) for k, v in model_map["HybridModelv2"](vae_input_dim=VAE_IN, device="cpu").state_dict().items()}
        sd = {k: torch.from_numpy(v).requires_grad_(True) for k, v in synthetic.det_state_dict(shapes, seed=3).items()}
        fine = self.finetune
        opt = torch.optim.Adam(list(sd.values()), lr=1e-4, weight_decay=1e-6) if fine else torch.optim.Adam(list(sd.values()), lr=1e-3)
        g = graph_ref.RefGraph(raw.src, raw.dst, raw.num_nodes, raw.batch_num_nodes)
        g.ndata["x"], g.edata["edge_attr"] = torch.from_numpy(raw.x), torch.from_numpy(raw.edge_attr)
        seq, prop = torch.from_numpy(raw.one_hot_sequence()), torch.from_numpy(raw.prop)
        y = torch.from_numpy(raw.y_bin if fine else raw.y_reg)

        def step():
            opt.zero_grad()
            it = FR.forward("HybridModelv2", sd, g, seq, prop)
            if fine:
                FR.bce_loss(it["recon_x"], seq, it["mu"], it["logvar"], it["final_output"], y, VAE_IN, 81.0 / 19.0).backward()
            else:
                FR.regression_loss(it["recon_x"], seq, it["mu"], it["logvar"], it["final_output"], y, VAE_IN).backward()
            opt.step()
        # the reference's per-step host work in front of the model (DataLoader: SplitDataset.__getitem__ deep-copies every
        # graph and rotates the copy's coordinates -- data/util_dataloader.py:27-29 -- then collate = dgl.batch + stack,
        # data/utils.py:160-176), restated on the oracle's graph type
        import copy
        n = int(raw.batch_num_nodes[0])
        order = np.argsort(raw.dst // n, kind="stable")
        bounds = np.concatenate([[0], np.cumsum(np.bincount(raw.dst // n, minlength=a.batch))])
        items = []
        for i in range(a.batch):
            e = order[bounds[i]:bounds[i + 1]]
            gi = graph_ref.RefGraph(raw.src[e] - i * n, raw.dst[e] - i * n, n)
            gi.ndata["x"], gi.edata["edge_attr"] = torch.from_numpy(raw.x[i * n:(i + 1) * n].copy()), torch.from_numpy(raw.edge_attr[e].copy())
            items.append((gi, seq[i].clone(), prop[i].clone(), y[i].clone()))

        def loader_step():
            nonlocal g, seq, prop, y
            samples = []
            for gi, si, pi, yi in items:
                c = copy.deepcopy(gi)
                q, _ = torch.linalg.qr(torch.randn(3, 3))
                c.ndata["x"][:, -3:] = c.ndata["x"][:, -3:] @ q
                samples.append((gi, si, pi, yi))      # (the reference hands the UN-rotated graph on: util_dataloader.py:82-86)
            graphs, seqs, props, ys = map(list, zip(*samples))
            g, seq, prop, y = graph_ref.batch(graphs), torch.stack(seqs), torch.stack(props), torch.stack(ys)
            step()
        return timed_cpu(step, a.batch, budget_s, f"B={a.batch} (oracle/functional_ref.py HybridModelv2, fwd+{'BCE' if fine else 'regression'} loss+bwd+Adam)",
                         loader_step=loader_step)


    def e2e(self, num_graphs=27000):
        """One epoch over a device-resident dataset of ``num_graphs`` synthetic graphs (the IEDB set's size, README.md:59) with
        the on-GPU batcher INSIDE the timed region: per step one gather launch from a shuffled id tensor into the captured
        step's static buffers + the replay (``procedures.train_model_device``'s inner loop)."""
        from immunostruct_amd.data import DeviceResidentDataset
        from immunostruct_amd.data.packed import PackedDataset
        from immunostruct_amd.engine import CapturedTrainStep
        a = self.args
        dev = next(self.model.parameters()).device
        t_build = time.perf_counter()
        raw = synthetic.make_batch(num_graphs, seed=77, deg_extra=a.deg_extra)
        n = int(raw.batch_num_nodes[0])
        counts = np.bincount(raw.dst // n, minlength=num_graphs)
        bounds = np.concatenate([[0], np.cumsum(counts)])
        order = np.argsort(raw.dst // n, kind="stable")
        src, dst, ea = raw.src[order], raw.dst[order], raw.edge_attr[order]
        graphs = [(raw.x[i * n:(i + 1) * n], torch.from_numpy(src[bounds[i]:bounds[i + 1]] - i * n),
                   torch.from_numpy(dst[bounds[i]:bounds[i + 1]] - i * n), torch.from_numpy(ea[bounds[i]:bounds[i + 1]]))
                  for i in range(num_graphs)]
        packed = PackedDataset.from_graphs(graphs, names=[str(i) for i in range(num_graphs)], pad_to=n)
        packed.seq, packed.prop = torch.from_numpy(raw.seq_tokens), torch.from_numpy(raw.prop)
        packed.y_reg, packed.y_bin = torch.from_numpy(raw.y_reg), torch.from_numpy(raw.y_bin)
        dds = DeviceResidentDataset.from_packed(packed, dev, binary=False)
        t_build = time.perf_counter() - t_build
        buf = dds.new_batch(a.batch)
        perm = torch.randperm(num_graphs, generator=torch.Generator().manual_seed(5)).to(dev)
        dds.gather_into(perm[:a.batch], *buf)
        eng = CapturedTrainStep(self.model, self.opt, D.FlatGradReducer(self.model.parameters(), world=1), self.forward_loss, buf,
                                edge_capacity=a.batch * dds.max_edges, warmup=1, step_random=STEP_RANDOM)
        steps = num_graphs // a.batch

        def epoch():
            for k in range(steps):
                dds.gather_into(perm[k * a.batch:(k + 1) * a.batch], eng.sgraph, eng.seq, eng.prop, eng.y)
                eng.replay()
        for k in range(5):
            dds.gather_into(perm[k * a.batch:(k + 1) * a.batch], eng.sgraph, eng.seq, eng.prop, eng.y)
            eng.replay()
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        epoch()
        torch.cuda.synchronize()
        dt = time.perf_counter() - t0
        return dict(value=round(steps * a.batch / dt, 1), unit="graphs/s", ms_per_step=round(1e3 * dt / steps, 3), steps=steps,
                    dataset_graphs=num_graphs, dataset_build_s=round(t_build, 1),
                    what="one epoch of full batches over a DeviceResidentDataset: shuffled ids -> on-GPU batcher (one gather launch "
                         "+ partition refresh) -> captured step replay, all inside the timed region (single GPU)")


class PairedWorkload(TrainStepWorkload):
    name = "paired"

    def __init__(self, args, dev, rank, world):
        from immunostruct_amd.graph import batch as graph_batch
        from immunostruct_amd.procedures.train import _paired_loss
        from immunostruct_amd.utils import PairedContrastiveLoss
        self.args, self.dev = args, dev
        self._paired_loss = _paired_loss
        torch.manual_seed(1)
        self.model = model_map["HybridModelv2_Comparative"](vae_input_dim=VAE_IN, device=dev, use_wt_for_downstream=True).to(dev)
        D.broadcast_parameters(self.model)
        self.model.train()
        self.opt = optim.AdamW(self.model.parameters(), lr=1e-4, weight_decay=1e-6)     # train_Cancer_wFT.py:76-92
        self.losses = Losses(VAE_IN, {0: 81.0, 1: 19.0}, sequence=True)
        self.contrastive = PairedContrastiveLoss(device=dev, embedding_dim=104)
        self.contrastive.capturable = True
        self.coeff = 0.01
        self.pool = []
        for i in range(3):
            rc = synthetic.make_batch(args.batch, seed=1000 * (rank + 1) + 10 + i, deg_extra=args.deg_extra)
            rw = synthetic.make_batch(args.batch, seed=1000 * (rank + 1) + 50 + i, deg_extra=args.deg_extra)
            bc, bw = device_batch(rc, dev, "y_bin"), device_batch(rw, dev, "y_bin")
            bc["g"].csr(), bw["g"].csr()
            # the merged pair batch [cancer; wild-type] the on-GPU batcher delivers (procedures.train_model_comparative_device)
            self.pool.append(dict(g=graph_batch([bc["g"], bw["g"]]), seq=torch.cat([bc["seq"], bw["seq"]]),
                                  prop=torch.cat([bc["prop"], bw["prop"]]), y=torch.cat([bc["y"], bc["y"]]),
                                  edges=rc.num_edges + rw.num_edges, nodes=rc.num_nodes + rw.num_nodes))
        self.graphs_per_step = 2 * args.batch
        self.n_nodes = self.pool[0]["nodes"]
        self.n_edges = float(np.mean([b["edges"] for b in self.pool]))
        self._finish(args, world, self.batch(0), max(b["edges"] for b in self.pool))

    def forward_loss(self, m, g2, seq2, prop2, y2):
        return self._paired_loss(m, self.losses.BCE_loss, (g2, seq2, y2[:y2.numel() // 2], prop2), self.dev, self.contrastive,
                                 self.coeff)
    forward_loss.fused_loss = True

    def batch(self, i):
        b = self.pool[i % len(self.pool)]
        return b["g"], b["seq"], b["prop"], b["y"]

    def describe(self):
        a = self.args
        return (f"cancer fine-tune step (BASELINE config 4): HybridModelv2_Comparative, use-wt-for-downstream, BCE + 0.01 x paired "
                f"contrastive loss, AdamW; B={a.batch} (cancer, wild-type) pairs = {2 * a.batch} graphs/GPU x 190 padded nodes, "
                f"E~{int(self.n_edges)} edges/step (deg_extra={a.deg_extra}), Fe=1; graphs/s counts both members")

    def roofline(self, timers, insitu=None):
        key = "paired_B128_deg2" if (self.args.batch == 128 and self.args.deg_extra == 2) else None
        return roofline_from_timers(timers, self.n_nodes, self.n_edges, (20, 64, 64, 64, 64), 1, key, insitu,
                                    paired_bwd=_paired_bwd_in_use(self.n_nodes, self.n_edges, 1))

    def cpu_baseline(self, budget_s=24.0):
        from oracle import functional_ref as FR
        from oracle import graph_ref
        a = self.args
        rc, rw = synthetic.make_batch(a.batch, seed=11, deg_extra=a.deg_extra), synthetic.make_batch(a.batch, seed=51, deg_extra=a.deg_extra)
        name = "HybridModelv2_Comparative"
        shapes = {k: tuple(v.shape) for k, v in model_map[name](vae_input_dim=VAE_IN, device="cpu").state_dict().items()}
        sd = {k: torch.from_numpy(v).requires_grad_(True) for k, v in synthetic.det_state_dict(shapes, seed=3).items()}
        proj = {k: torch.from_numpy(v) for k, v in synthetic.det_state_dict(
            {"projector.0.weight": (128, 104), "projector.1.weight": (128,), "projector.1.bias": (128,),
             "projector.3.weight": (128, 128)}, seed=9).items()}
        opt = torch.optim.AdamW(list(sd.values()), lr=1e-4, weight_decay=1e-6)

        def ref_graph(raw):
            g = graph_ref.RefGraph(raw.src, raw.dst, raw.num_nodes, raw.batch_num_nodes)
            g.ndata["x"], g.edata["edge_attr"] = torch.from_numpy(raw.x), torch.from_numpy(raw.edge_attr)
            return g
        gs = (ref_graph(rc), ref_graph(rw))
        seqs = (torch.from_numpy(rc.one_hot_sequence()), torch.from_numpy(rw.one_hot_sequence()))
        props = (torch.from_numpy(rc.prop), torch.from_numpy(rw.prop))
        y = torch.from_numpy(rc.y_bin)

        def step():
            opt.zero_grad()
            o = FR.forward_comparative(name, sd, gs, seqs, props)
            c, w = o["cancer"], o["wt"]
            lc = FR.bce_loss(c["recon_x"], seqs[0], c["mu"], c["logvar"], o["final_output"], y, VAE_IN, 81.0 / 19.0)
            lw = FR.bce_loss(w["recon_x"], seqs[1], w["mu"], w["logvar"], o["final_output"], y, VAE_IN, 81.0 / 19.0)
            loss = (lc + lw) / 2 + 0.01 * FR.paired_contrastive_loss(proj, o["embeddings"][0], o["embeddings"][1], y)
            loss.backward()
            opt.step()
        return timed_cpu(step, 2 * a.batch, budget_s,
                         f"B={a.batch} pairs (oracle/functional_ref.py forward_comparative + BCE + paired contrastive, fwd+bwd+AdamW)")


STRESS_N_MIN, STRESS_N_MAX = 155, 245


def stress_batch(num_graphs, seed):
    """config 5: node counts ~ N(200, 15) clipped to [155, 245] and padded to 245, 8 edge features ~ U(0, 1), chain + 7
    random contacts per node (average in-degree 8)"""
    choices = np.arange(STRESS_N_MIN, STRESS_N_MAX + 1)
    w = np.exp(-0.5 * ((choices - 200.0) / 15.0) ** 2)
    return synthetic.make_batch(num_graphs, seed=seed, n_pad=STRESS_N_MAX, deg_extra=7, edge_feats=8,
                                n_real_choices=tuple(int(c) for c in choices), n_real_probs=tuple(float(v) for v in w / w.sum()))


class StressWorkload:
    name = "stress"
    LAYERS = 6
    # config 5 is a kernel stress of the graph encoder: the reference's model classes hard-code edge_feat_size = 1
    # (models/hybrid_models.py:29), so no train step with 8 edge features exists to time
    metric = "residue graphs/sec (EGNN stack forward + backward, no heads, no optimizer)"

    def __init__(self, args, dev, rank, world):
        from immunostruct_amd.nn import EGNNConv, egnn_stack_forward
        self.args, self.dev = args, dev
        self._stack = egnn_stack_forward
        torch.manual_seed(1)
        self.layers = torch.nn.ModuleList([EGNNConv(H, H, H, 8) for _ in range(self.LAYERS)]).to(dev)
        D.broadcast_parameters(self.layers)
        self.reducer = D.FlatGradReducer(self.layers.parameters(), world=world, always_pack=args.force_pack)
        gen = torch.Generator().manual_seed(7 + rank)
        self.pool = []
        for i in range(3):
            raw = stress_batch(args.batch, seed=2000 * (rank + 1) + i)
            g = PackedGraphBatch.from_raw(raw, device=dev)
            g.csr()
            n = raw.num_nodes
            self.pool.append(dict(g=g, raw=raw, h0=(0.5 * torch.randn(n, H, generator=gen)).to(dev),
                                  x0=torch.from_numpy(raw.x[:, 20:].copy()).to(dev),
                                  gh=(torch.randn(n, H, generator=gen) / n).to(dev), gx=(torch.randn(n, 3, generator=gen) / n).to(dev)))
        self.graphs_per_step = args.batch
        self.n_nodes = self.pool[0]["raw"].num_nodes
        self.n_edges = float(np.mean([b["raw"].num_edges for b in self.pool]))
        self.graphs = None
        if not args.eager:
            # one captured HIP graph per resident batch (the batches differ in edge count; nothing is copied per step)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for i in range(len(self.pool)):
                    self._body(i)
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            self.graphs = []
            for i in range(len(self.pool)):
                gr = torch.cuda.CUDAGraph()
                with torch.cuda.graph(gr, capture_error_mode="thread_local"):      # (a process group's watchdog thread polls events)
                    self._body(i)
                self.reducer.bind_sources()
                self.graphs.append((gr, self.reducer.sources()))

    def _body(self, i):
        b = self.pool[i]
        self.reducer.zero()
        h, x = self._stack(list(self.layers), b["g"], b["h0"], b["x0"], b["g"].edata["edge_attr"])
        torch.autograd.backward([h, x], [b["gh"], b["gx"]])

    def step(self, i):
        if self.graphs is None:
            return self.eager_step(i)
        gr, srcs = self.graphs[i % len(self.pool)]
        gr.replay()
        if self.reducer.packing:
            self.reducer.sources(srcs)
            self.reducer.all_reduce_mean()
        return None

    def eager_step(self, i):
        for bucket in self.reducer.buckets:
            bucket["sources"] = None
        self._body(i % len(self.pool))
        if self.reducer.packing:
            self.reducer.all_reduce_mean()
        return None

    def eager_timers_setup(self):
        return lambda: None

    def describe(self):
        a = self.args
        return (f"EGNN-stack stress (BASELINE config 5, one GPU's slice): {self.LAYERS} EGNNConv layers (64 -> 64 channels, 8 edge "
                f"features) forward + backward with all weight gradients, no optimizer; B={a.batch} graphs/GPU, node counts "
                f"~N(200,15) clipped to [{STRESS_N_MIN},{STRESS_N_MAX}] padded to {STRESS_N_MAX}, N={self.n_nodes} nodes, "
                f"E~{int(self.n_edges)} edges/step (average in-degree 8)")

    def extra_config(self):
        return dict(launch="eager" if self.graphs is None else "hipGraph replay",
                    grad_allreduce=None if not self.reducer.packing else
                    dict(form="serial", buckets=[int(b["flat"].numel()) for b in self.reducer.buckets]))

    def roofline(self, timers, insitu=None):
        key = "stress_B256" if self.args.batch == 256 else None
        return roofline_from_timers(timers, self.n_nodes, self.n_edges, (64,) * self.LAYERS, 8, key, insitu)

    def cpu_baseline(self, budget_s=24.0):
        from oracle import graph_ref
        b = min(self.args.batch, 32)
        raw = stress_batch(b, seed=1)
        shapes = {}
        for i in range(self.LAYERS):
            p = f"L{i}."
            shapes.update({p + "edge_mlp.0.weight": (H, 2 * H + 1 + 8), p + "edge_mlp.0.bias": (H,), p + "edge_mlp.2.weight": (H, H),
                           p + "edge_mlp.2.bias": (H,), p + "node_mlp.0.weight": (H, 2 * H), p + "node_mlp.0.bias": (H,),
                           p + "node_mlp.2.weight": (H, H), p + "node_mlp.2.bias": (H,), p + "coord_mlp.0.weight": (H, H),
                           p + "coord_mlp.0.bias": (H,), p + "coord_mlp.2.weight": (1, H)})
        sd = {k: torch.from_numpy(v).requires_grad_(True) for k, v in synthetic.det_state_dict(shapes, seed=3).items()}
        src, dst = torch.from_numpy(raw.src), torch.from_numpy(raw.dst)
        gen = torch.Generator().manual_seed(7)
        n = raw.num_nodes
        h0, x0 = 0.5 * torch.randn(n, H, generator=gen), torch.from_numpy(raw.x[:, 20:].copy())
        gh, gx = torch.randn(n, H, generator=gen) / n, torch.randn(n, 3, generator=gen) / n
        ea = torch.from_numpy(raw.edge_attr)

        def step():
            for v in sd.values():
                v.grad = None
            h, x = h0, x0
            for i in range(self.LAYERS):
                h, x = graph_ref.egnn_conv(sd, f"L{i}.", src, dst, n, h, x, ea)
            torch.autograd.backward([h, x], [gh, gx])
        return timed_cpu(step, b, budget_s, f"B={b} graphs of the same distribution (oracle/graph_ref.py egnn_conv x {self.LAYERS}, fwd+bwd)")


WORKLOADS = {"iedb": IedbWorkload, "paired": PairedWorkload, "stress": StressWorkload}


def flush_c_stdio():
    """libraries (RCCL) print through libc's buffered stdout, which would otherwise be flushed at exit -- AFTER the one
    JSON line this script promises as its last output"""
    import ctypes
    sys.stdout.flush()
    try:
        ctypes.CDLL(None).fflush(None)
    except OSError:
        pass


def self_launch(n):
    """``python bench.py --gpus N`` without torchrun: start one child per GPU (RANK / LOCAL_RANK / WORLD_SIZE / MASTER_*
    in its environment, the contract torch.distributed.run would provide) BEFORE this process touches a GPU, let rank 0
    write the single JSON line to our stdout (the other ranks' stdout goes to stderr), and return non-zero when any
    rank fails -- the survivors are then stopped by PID, never by pattern."""
    import socket
    import subprocess
    have = torch.cuda.device_count()       # counting devices does not initialise the GPU runtime
    if have < n and os.environ.get("IMMUNOSTRUCT_FORCE_DEVICE") is None:
        print(f"bench.py: --gpus {n} requested but {have} GPU(s) visible", file=sys.stderr)
        return 2
    env = dict(os.environ)
    env.setdefault("MASTER_ADDR", "127.0.0.1")
    if "MASTER_PORT" not in env:
        with socket.socket() as so:
            so.bind(("127.0.0.1", 0))
            env["MASTER_PORT"] = str(so.getsockname()[1])
    env.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")
    env["WORLD_SIZE"] = env["LOCAL_WORLD_SIZE"] = str(n)
    procs = []
    for r in range(n):
        e = dict(env, RANK=str(r), LOCAL_RANK=str(r))
        procs.append(subprocess.Popen([sys.executable, os.path.abspath(__file__)] + sys.argv[1:], env=e,
                                      stdout=None if r == 0 else sys.stderr))
    rc, pending = 0, set(range(n))
    while pending:
        for r in sorted(pending):
            code = procs[r].poll()
            if code is None:
                continue
            pending.discard(r)
            if code != 0 and rc == 0:
                rc = code if code > 0 else 1
                print(f"bench.py: rank {r} exited with {code}; stopping the other ranks", file=sys.stderr)
                for q in sorted(pending):
                    procs[q].terminate()
        time.sleep(0.05)
    return rc


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--warmup", type=int, default=5)
    # (the driver runs the plain command line: IMMUNOSTRUCT_BENCH_WORKLOAD / IMMUNOSTRUCT_BENCH_STAGE select another line)
    ap.add_argument("--workload", choices=sorted(WORKLOADS), default=os.environ.get("IMMUNOSTRUCT_BENCH_WORKLOAD", "iedb"))
    ap.add_argument("--stage", choices=("pretrain", "finetune"), default=os.environ.get("IMMUNOSTRUCT_BENCH_STAGE", "pretrain"),
                    help="iedb: regression stage (Adam 1e-3) or the BCE finetune stage (Adam 1e-4, weight decay 1e-6)")
    ap.add_argument("--batch", type=int, default=None, help="graphs (paired: pairs) per GPU per step; default 128 (stress: 256)")
    ap.add_argument("--deg-extra", type=int, default=2, help="iedb / paired: random contact edges per residue (E/N - 1)")
    ap.add_argument("--symmetric-edges", action="store_true", help="iedb: every chain link / contact in both directions (2 x the edges)")
    ap.add_argument("--model", default="HybridModelv2", help="iedb: the model class")
    ap.add_argument("--no-cpu-baseline", action="store_true")
    ap.add_argument("--no-e2e", action="store_true", help="iedb, one GPU: skip the batcher-inclusive epoch over 27 000 resident graphs")
    ap.add_argument("--no-host-read", action="store_true", help="skip the step_with_host_read sample (profiled runs: the last step of the trace stays a plain replay)")
    ap.add_argument("--e2e-graphs", type=int, default=27000)
    ap.add_argument("--no-kernel-timers", action="store_true")
    ap.add_argument("--no-copy-ceiling", action="store_true", help="skip the measured device-to-device copy bandwidth (2 x 1 GiB)")
    ap.add_argument("--force-pack", action="store_true", help="exercise the multi-rank gradient-bucket path on one GPU")
    ap.add_argument("--eager", action="store_true", help="launch every kernel eagerly instead of replaying the captured HIP graph")
    args = ap.parse_args()
    if args.batch is None:
        args.batch = 256 if args.workload == "stress" else 128

    if args.gpus > 1 and "WORLD_SIZE" not in os.environ:
        # started as plain ``python bench.py --gpus N``: become the launcher (no GPU call has happened in this process)
        raise SystemExit(self_launch(args.gpus))
    rank, local_rank, world = D.init_from_env()
    if world != args.gpus:
        raise SystemExit(f"--gpus {args.gpus} but WORLD_SIZE={world}: the line printed must describe the run asked for")
    if not torch.cuda.is_available():
        raise SystemExit("bench.py needs a ROCm GPU (the product path has no CPU fallback)")
    if os.environ.get("IMMUNOSTRUCT_FORCE_DEVICE") is not None:   # debugging aid: several ranks on one GPU (gloo)
        local_rank = int(os.environ["IMMUNOSTRUCT_FORCE_DEVICE"])
    torch.cuda.set_device(local_rank)
    dev = torch.device("cuda", local_rank)

    # in-situ launch timing of the layer kernels (workgroup clocks; functional.LaunchClock): the buffers must exist before the
    # step is captured, and cost two 8-byte stores per workgroup
    HF.LaunchClock.enabled = not args.no_kernel_timers
    wl = WORKLOADS[args.workload](args, dev, rank, world)
    step = wl.step

    def fence():
        if world > 1:
            torch.distributed.barrier()
        torch.cuda.synchronize()

    for i in range(args.warmup):
        step(i)
    # (everything that takes host time without GPU work -- the collector pass, the creation of the timing events -- happens HERE,
    #  in front of the settle blocks: between the last settle block and the timed region the GPU must not sit idle, or the timed
    #  steps start on a device that has dropped its clocks: 15 steps of ramp, +2 % on a 30-step mean)
    gc.collect()
    gc.disable()          # no collector pause inside the (tens of milliseconds long) timed region
    marks = [torch.cuda.Event(enable_timing=True) for _ in range(args.steps + 1)]
    flush_c_stdio()       # RCCL's version banner sits in libc's stdout buffer: push it out now, not after the JSON line
    # untimed: keep replaying until the step time is stable (clocks / caches / allocator of a cold box), at most ~0.5 s;
    # every rank runs the same number of blocks (the stop decision is rank 0's)
    settle, prev = [], None
    fixed_blocks = os.environ.get("IMMUNOSTRUCT_BENCH_SETTLE_BLOCKS")      # tests: a run-to-run identical number of steps
    for blk in range(40 if fixed_blocks is None else int(fixed_blocks)):
        fence()
        s0 = time.perf_counter()
        for i in range(5):
            step(args.warmup + i)
        fence()
        cur = (time.perf_counter() - s0) / 5
        settle.append(round(cur * 1e3, 3))
        stop = fixed_blocks is None and ((prev is not None and abs(cur - prev) <= 0.02 * prev and blk >= 2) or sum(settle) * 5e-3 > 0.5)
        if world > 1:
            flag = torch.tensor([1 if stop else 0], device=dev)
            torch.distributed.broadcast(flag, src=0)
            stop = bool(flag.item())
        if stop:
            break
        prev = cur
    HF.KernelTimer.reset()
    HF.KernelTimer.enabled = args.eager and not args.no_kernel_timers
    fence()
    t0 = time.perf_counter()
    last = None
    for i in range(args.steps):
        marks[i].record()
        last = step(args.warmup + i)
    marks[args.steps].record()
    fence()
    dt = time.perf_counter() - t0
    gc.enable()
    HF.KernelTimer.enabled = False
    per_step = [a.elapsed_time(b) for a, b in zip(marks, marks[1:])]      # device time between the steps' first launches
    if os.environ.get("IMMUNOSTRUCT_BENCH_STEP_TRACE"):      # debugging aid: the timed steps in order (which ones are slow?)
        print("[step trace ms] " + " ".join(f"{v:.3f}" for v in per_step), file=sys.stderr)
    per_step = sorted(per_step)
    # the reference's loop reads the loss back on the host every step (procedures/train.py:29 ``loss.item()``): the same replay with
    # that read, outside the timed region -- the host then waits for every step before it enqueues the next one
    host_read = None
    if not args.eager and not args.no_host_read:
        n_hr = min(args.steps, 20)
        fence()
        h0 = time.perf_counter()
        acc = 0.0
        for i in range(n_hr):
            l = step(args.warmup + i)
            if l is not None:
                acc += float(l)                     # .item(): a device -> host copy and a synchronisation per step
            else:
                torch.cuda.synchronize()            # (a workload without a loss: the synchronisation alone)
        fence()
        hdt = time.perf_counter() - h0
        if world > 1:
            t = torch.tensor([hdt], dtype=torch.float64, device=dev)
            D.all_reduce(t, op=torch.distributed.ReduceOp.MAX)
            hdt = float(t.item())
        host_read = dict(steps=n_hr, ms_per_step=round(hdt / n_hr * 1e3, 3), mean_loss=round(acc / n_hr, 6),
                         note="the same replayed step followed by float(loss) on the host, as the reference's loop does "
                              "(procedures/train.py:29); `value` is the device-throughput figure without that read")
    if os.environ.get("IMMUNOSTRUCT_HOST_TIMES"):     # debugging aid: host-side cost of one isolated step vs its GPU time
        for i in range(5):
            fence()
            h0 = time.perf_counter()
            step(args.warmup + args.steps + i)
            h1 = time.perf_counter()
            fence()
            h2 = time.perf_counter()
            print(f"[host times] step call returned after {1e6 * (h1 - h0):.0f} us, GPU done after {1e6 * (h2 - h0):.0f} us", file=sys.stderr)
    if HF.Stamps.enabled and HF.Stamps.buf is not None:
        fence()
        for t_us, name in HF.Stamps.report():
            print(f"[stamps] {t_us:9.1f} us  {name}", file=sys.stderr)
    if world > 1:
        t = torch.tensor([dt], dtype=torch.float64, device=dev)
        D.all_reduce(t, op=torch.distributed.ReduceOp.MAX)
        dt = float(t.item())
    final_loss = float(last.detach()) if last is not None else None
    insitu = None
    if HF.LaunchClock.enabled:
        # the replayed graph's launches stamp their workgroups' start / end clocks on every replay: sample a few more replays of
        # the SAME graph(s) the timed region ran (every rank steps -- the step may hold a collective; rank 0 reads the clocks back
        # after each replay; outside the timed region)
        insitu = {}
        for i in range(min(args.steps, 12)):
            step(args.warmup + i)
            torch.cuda.synchronize()
            if rank == 0:
                for kind, d in HF.LaunchClock.durations().items():
                    ent = insitu.setdefault(kind, {"span": [], "slot": []})
                    ent["span"] += d["span"]
                    ent["slot"] += d["slot"]
    timers_mode = "HIP events around each launch inside the timed region (eager launches)"
    if not args.eager and not args.no_kernel_timers:
        # the timed region replays a captured HIP graph (individual launches cannot be bracketed there): measure per-kernel
        # durations with HIP events on an eager re-run of the same steps (the in-situ averages are in profiles/)
        restore = wl.eager_timers_setup()
        for i in range(2):      # untimed: the first eager steps after the replays grow the allocator's pool (hipMalloc stalls)
            wl.eager_step(args.warmup + i)
        torch.cuda.synchronize()
        HF.KernelTimer.reset()
        HF.KernelTimer.enabled = True
        # the layer kernels (the roofline's subject; idempotent) are issued 4 x back to back inside ONE event pair: on an idle
        # GPU a pair also brackets the host's launch latency (~10 us), which 4 launches pay once; and from the second launch
        # on the kernel runs as it does inside the replayed step (GPU busy, no gap in front)
        HF.KernelTimer.repeat = 4
        HF.KernelTimer.repeat_names = frozenset(("egnn_layer_fwd", "egnn_layer_fwd_nocoord", "egnn_layer_bwd", "egnn_layer_bwd_nocoord"))
        for i in range(min(args.steps, 10)):
            wl.eager_step(args.warmup + i)
        torch.cuda.synchronize()
        HF.KernelTimer.enabled = False
        HF.KernelTimer.repeat, HF.KernelTimer.repeat_names = 1, frozenset()
        restore()
        timers_mode = ("HIP events on the launching stream, eager single-stream re-run of the timed steps (the timed region replays a "
                       "HIP graph, where a launch cannot be bracketed); the two layer kernels are issued 4 x back to back inside one "
                       "event pair (duration / 4), every other kernel once per pair")

    extra_config = wl.extra_config()      # every rank: it times the standalone all-reduce of the buckets (collectives)
    if rank == 0:
        graphs = wl.graphs_per_step * world * args.steps
        timers = HF.KernelTimer.summary()
        roof = wl.roofline(timers, insitu)
        if roof is not None:
            roof["eager_us_measured"] = timers_mode
            if insitu:
                st = lambda v: dict(mean=round(float(np.mean(v)), 2), min=round(float(np.min(v)), 2), max=round(float(np.max(v)), 2),
                                    samples=len(v)) if v else None
                roof["insitu_us"] = {k: dict(slot=st(v["slot"]), span=st(v["span"])) for k, v in sorted(insitu.items())}
        ceiling = None
        if not args.no_copy_ceiling:
            ceiling = measured_copy_ceiling(dev)
            attach_measured_peak(roof, ceiling)
        cpu = e2e = None
        if world == 1 and not args.no_e2e and not args.eager and hasattr(wl, "e2e"):
            e2e = wl.e2e(args.e2e_graphs)
        if world == 1 and not args.no_cpu_baseline:
            cpu = wl.cpu_baseline()
        ddp = torch.distributed.is_initialized()
        config = dict(workload=wl.describe(), global_batch=wl.graphs_per_step * world, nodes_per_batch=wl.n_nodes,
                      edges_per_batch=int(wl.n_edges), parallelism=f"dp{world}",
                      final_loss=None if final_loss is None else round(final_loss, 7),
                      rccl_ranks=torch.distributed.get_world_size() if ddp else 1,
                      dist_backend=torch.distributed.get_backend() if ddp else None,
                      # operators that left the HIP kernels' build for a device-side torch composition (functional.composed_path):
                      # {} = every operator of the timed step ran on the hand-written kernels
                      composed_paths=dict(HF.COMPOSED_PATHS))
        config.update(extra_config)
        if host_read is not None:
            host_read["value"] = round(wl.graphs_per_step * world / (host_read["ms_per_step"] * 1e-3), 1)
            host_read["unit"] = "graphs/s"
        if roof is not None and "hbm_view" in roof:
            # the figures BASELINE.json's metric names ("GNN-gather achieved HBM GB/s", ">= 40 % of the HBM roofline on the gather /
            # scatter kernel"), plainly, beside the MFMA fraction the dominant kernel is bounded by: fractions of the 8 TB/s SPEC
            roof["hbm_frac"] = roof["hbm_view"]["frac"]      # dominant (fused layer backward) kernel, algorithmic bytes / slot time
            gk = roof.get("gather_kernel")
            if gk is not None:
                roof["gather_frac"] = gk["frac"]              # the residual pure gather launch (layer 0), algorithmic bytes / slot time
                span = (roof.get("insitu_us", {}).get("gather") or {}).get("span")
                if span:
                    gb = gk["achieved"] * gk["mean_launch_us"] * 1e-6      # GB per launch
                    gk["span_us"] = span["mean"]
                    gk["achieved_over_span"] = round(gb / (span["mean"] * 1e-6), 1)
                    gk["frac_over_span"] = round(gb / (span["mean"] * 1e-6) / PEAK_HBM_GBS, 4)
            # the contract, said once (DESIGN.md 4.1 "Roofline accounting"): which bound each number is priced against, and what became
            # of the north star's HBM target
            roof["contract"] = (
                "frac = algorithmic FLOP of the dominant kernel (the fused EGNN layer backward: gather + edge / coordinate / node MLP "
                "backward + segment sums in ONE launch, ~65 FLOP per algorithmic byte against a ridge of 157.3 TFLOP/s / 8 TB/s = "
                "19.7 FLOP/B) / its slot time / the dense fp32 MFMA peak: the kernel is MFMA- (instruction-issue-) bound, `bound` says "
                "so, and this is the fraction it is judged by.  hbm_frac = the SAME launch's algorithmic bytes / slot time / 8 TB/s: "
                "reported because BASELINE.json's metric names HBM GB/s, NOT a target of the fused kernel -- fusing the per-edge "
                "arithmetic into the gather is what removes its bytes.  The north star's '>= 40 % of the HBM roofline on the gather / "
                "scatter kernel' applies to what is left as a pure gather, gather_segment_sum (layer 0's scatter-add to source rows, "
                "one launch per step): gather_frac, by slot time -- NOT met at this batch size (a 26 MB launch lasts three dependent "
                "round trips + the dispatch gap whatever its kernel does; gather_kernel.frac_over_span is the launch alone).")
        line = dict(metric=getattr(wl, "metric", "peptide-MHC graphs/sec (train step)"), value=round(graphs / dt, 1), unit="graphs/s",
                    n_gpus=world, steps=args.steps, warmup=args.warmup, ms_per_step=round(dt / args.steps * 1e3, 3),
                    higher_is_better=True, scaling="weak", vs_baseline=None, dtype="f32", data="synthetic", config=config,
                    step_ms=dict(median=round(per_step[len(per_step) // 2], 3), min=round(per_step[0], 3), max=round(per_step[-1], 3),
                                 settle_blocks_ms=settle,
                                 note="device time per step from HIP events between the steps (rank 0); settle_blocks_ms = the "
                                      "untimed 5-step blocks replayed after the warm-up until two agreed within 2 %"),
                    step_with_host_read=host_read, roofline=roof, hbm_copy_ceiling=ceiling, cpu_baseline=cpu, e2e=e2e,
                    kernel_timers_us={k: [v[0], round(v[1] * 1e3, 2)] for k, v in timers.items()})
        flush_c_stdio()
        print(json.dumps(line), flush=True)
    if torch.distributed.is_initialized():
        # teardown in dependency order: the captured graphs (which may hold RCCL's collective nodes) go first, then the process group --
        # destroying the communicator under a live graph that references it aborted one run in a dozen on the one-rank RCCL group
        torch.cuda.synchronize()
        if getattr(wl, "captured", None) is not None:
            wl.captured.close()
        for name in ("captured", "graphs"):
            if hasattr(wl, name):
                setattr(wl, name, None)
        gc.collect()
        torch.cuda.synchronize()
        if world > 1:
            torch.distributed.barrier()
        torch.distributed.destroy_process_group()


if __name__ == "__main__":
    main()
