"""G7 on the GPU: the full training forward/backward with the HIP kernels in the loop reproduces
the reference's losses / poses / gradients recorded in tests/golden/step_*.npz.

Tolerances: north_star's 1e-4 relative on every loss scalar and on the predicted pose.  Gradients:
cosine >= 0.9998 and relative L2 <= 3e-2 (observed over runs: mean_v 0.99992-0.99998 / 0.6-1.2e-2,
every other probe >= 0.99998 / <= 5e-3; MIOpen's solver search makes runs differ) -- the band two legal builds of the reference's own kernels
exhibit (SURVEY F12 iii): MIOpen/rocBLAS round the encoder outputs differently from the CPU
(poses differ by ~5e-6), and the gamma=1e-4 depth softmax amplifies such input perturbations in
individual gradient elements.  On IDENTICAL inputs the HIP kernels agree with the oracle to 1e-4 of
the gradient scale (tests/test_softras_gpu.py)."""
import pytest
import torch

import step_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", ["step_laptopflags_bottle_b2x2", "step_laptopflags_laptop_b2x2",
                                  "step_laptopflags_bottle_b1x1"])
def test_full_step_matches_reference_on_gpu(case):
    """strict: encoder geometry pinned to the reference's values (see step_case.pin_encoder_geometry),
    everything downstream -- correspondence, 4 render passes, DINO cycle, all losses, backward --
    runs on the HIP kernels; every loss within north_star's 1e-4 relative"""
    model, data, d = step_case.build("cuda", case)
    from scp_amd.soft_renderer.cuda import soft_rasterize as native
    assert native.forward_soft_rasterize.__module__.startswith("scp_amd"), "HIP path must be the one that runs"
    step_case.pin_encoder_geometry(model, d)
    report = step_case.run_and_compare(model, data, d, grad_rel_l2=3e-2, grad_cos=0.9998)
    report["nn_flip_fraction"] = step_case.check_mutual_nn_validity(model, d)
    print({k: v for k, v in report.items()})


def test_full_step_free_running_on_gpu():
    """nothing pinned but the discrete selections.  The stock MIOpen/rocBLAS encoder rounds pred_v / pose
    differently from the CPU reference (measured and asserted below: <= 1e-5), and the silhouette-sensitive render
    terms amplify that.  The allowed deviation per loss is NOT hand-picked: it is the spread the REFERENCE ITSELF shows
    when its own encoder outputs are perturbed at that level (tests/golden/step_conditioning_bottle_b2x2.npz, recorded by
    make_golden.py step_conditioning; see step_case.conditioning_band).  Terms the reference holds to 1e-4 under such
    perturbations must meet north_star's 1e-4 here.  (Round 3 asserted min(band, 3 x the largest deviation this build had shown so
    far); that self-calibrated table is gone and tools/parity_sweep.py (profiles/r04_parity_sweep.txt) shows the
    free-running deviations do not depend on which matrix cores the encoder / ViT run on.)"""
    import numpy as np
    model, data, d = step_case.build("cuda")
    band, spread, sigmas = step_case.conditioning_band("step_conditioning_bottle_b2x2")
    cap = {}
    fwd = model.encoder.forward

    def spy(*a, **k):
        out = fwd(*a, **k)
        cap["enc"] = out
        return out
    model.encoder.forward = spy
    report = step_case.run_and_compare(model, data, d, rtol_loss=band, grad_rel_l2=0.1, grad_cos=0.995)
    # the premise of the band: the encoder's geometric outputs deviate from the reference's by no more than the
    # perturbation levels the fixture covers
    for j, key in ((2, "pred_v"), (3, "rotation"), (4, "translation")):
        dev = np.abs(cap["enc"][j].detach().cpu().numpy().astype(np.float64) - d[key])
        print("encoder %-12s deviation from the reference: rms %.2e max %.2e" % (key, np.sqrt((dev ** 2).mean()), dev.max()))
        assert np.sqrt((dev ** 2).mean()) <= float(sigmas.max())
    # the assertion itself is run_and_compare's (rtol_loss = the reference-recorded band, nothing derived from this build's own
    # observations); the table is for the log
    for k, (got, ref) in report.items():
        if k in band:
            print("%-22s rel dev %.2e | band %.2e = max(1e-4, 1.5 x the reference's own spread under perturbation %.2e)"
                  % (k, abs(got - ref) / max(abs(ref), 1e-12), band[k], spread[k]))


def test_full_step_b8_laptop_vs_oracle_backend(monkeypatch):
    """BASELINE configs[1] as a WHOLE step (B = 8 = batch_size 2 x repeat 4, laptop mesh 995 v / 1986 f): forward + backward on
    the GPU (HIP kernels) against the same step on the CPU oracle backend (oracle/backend.py: C rasteriser + torch
    restatements, themselves pinned to the reference's recordings in tests/golden).  Identical recipe weights, batch and
    pinned RNG consumers; the CPU side's mutual-NN / top-k selections are injected on the GPU side.
    Every loss term within max(1e-4, the reference's own conditioning band), poses within 1e-4 / 1e-5, probe gradients
    cos >= 0.9995 / rel-L2 <= 5e-2."""
    import numpy as np
    import golden_io
    import oracle_backend
    import recipe
    import synth
    import scp_amd.dino as dino
    from scp_amd.flags import Options
    from scp_amd.model import MeshNet
    d = golden_io.load("step_laptopflags_laptop_b2x2")
    assert d["prior_verts"].shape[0] == 995 and d["prior_faces"].shape[0] == 1986
    dino.ALLOW_RANDOM_INIT = True
    bs, rep = 2, 4

    def build(device):
        opts = Options("laptop_wild6d", batch_size=bs, repeat=rep, train=True, vis_freq=10 ** 9)
        torch.manual_seed(0)
        model = MeshNet(opts, prior=(d["prior_verts"], d["prior_faces"]))
        recipe.load_recipe(model)
        model.encoder.random_jitter = torch.nn.Identity()
        model.rotation_angle = 90.0
        k = model.mesh.symm_rots.shape[0]
        fi, bary = recipe.symmetry_sample(k * bs * rep, 10000, model.mesh.num_faces)
        model = model.to(device).train()
        model.mesh.sample_override = (fi.to(device), bary.to(device))
        model.iters = 0
        return model

    probes = {"mean_v": "mesh.mean_v", "resnet_conv1": "encoder.backbone.resnet.conv1.weight", "featnet_proj": "encoder.featnet.proj.weight",
              "pose_trans": "encoder.pose_predictor.trans_pred_layer.weight", "mesh_stn_fc": "encoder.featnet_mesh.stn.fc.weight"}

    def run(model, data):
        total, aux = model(data)
        total.mean().backward()
        params = dict(model.named_parameters())
        return ({k: float(v) for k, v in aux.items()}, [t.detach().cpu().double().numpy() for t in model.last_pose],
                {k: params[n].grad.detach().cpu().double().numpy().ravel() for k, n in probes.items()})

    with monkeypatch.context() as mp:
        oracle_backend.install(mp)                     # CPU stand-ins for every HIP kernel (checker side only)
        cpu = build("cpu")
        ref_aux, ref_pose, ref_grad = run(cpu, synth.make_batch(bs, rep, 256, seed=3, device="cpu"))
        pc = cpu.pretrain_corr_net
        sel_nn, sel_topk = tuple(t.clone() for t in pc.last_nn), pc.last_topk.clone()
    gpu = build("cuda")
    from scp_amd.soft_renderer.cuda import soft_rasterize as native
    assert native.forward_soft_rasterize.__module__.startswith("scp_amd"), "HIP path must be the one that runs"
    gpu.pretrain_corr_net.nn_override = tuple(t.cuda() for t in sel_nn)
    gpu.pretrain_corr_net.topk_override = sel_topk.cuda()
    got_aux, got_pose, got_grad = run(gpu, synth.make_batch(bs, rep, 256, seed=3, device="cuda"))
    band, _, _ = step_case.conditioning_band("step_conditioning_laptop_b2x4")     # recorded from the reference at this mesh / batch
    for k, ref in ref_aux.items():
        rel = abs(got_aux[k] - ref) / max(abs(ref), 1e-6)
        print("%-22s cpu-oracle %.9g gpu %.9g rel %.2e" % (k, ref, got_aux[k], rel))
        assert rel <= band.get(k, 1e-4), "%s: %.9g vs %.9g (rel %.2e)" % (k, got_aux[k], ref, rel)
    # poses: 1e-4 relative to the quantity's scale -- a rotation matrix has unit rows (entries near zero cannot be compared
    # relatively; observed: <= 2.3e-5 absolute in the full-suite process, ~1e-5 alone), translations are O(1)
    np.testing.assert_allclose(got_pose[0], ref_pose[0], rtol=1e-4, atol=5e-5)
    np.testing.assert_allclose(got_pose[1], ref_pose[1], rtol=1e-4, atol=5e-5)
    for k in probes:
        g, r = got_grad[k], ref_grad[k]
        rel = np.linalg.norm(g - r) / np.linalg.norm(r)
        cos = g @ r / (np.linalg.norm(g) * np.linalg.norm(r))
        print("grad %-14s rel L2 %.3e cos %.7f" % (k, rel, cos))
        assert rel <= 5e-2 and cos >= 0.9995, "%s: rel L2 %.3e cos %.7f" % (k, rel, cos)


def test_full_step_b32_headline_config_vs_oracle_backend(monkeypatch):
    """BASELINE configs[2] -- the bench workload itself -- as a WHOLE step inside the suite: B = 32 (batch_size 8 x repeat 4), 256 x 256,
    bottle mesh 642 v / 1280 f, laptop flags; forward + backward on the GPU (HIP kernels, the shipped stream schedule) against the same
    step on the CPU oracle backend (model/trainer.py:118-125's forward/backward).  Identical weights (seed 0 on the host), batch, pinned
    RNG consumers; the CPU side's mutual-NN / top-k selections injected.  Two legs, as bench.py's loss_delta:
      pinned        the encoder's outputs take the CPU side's values (autograd path kept): every loss term <= 1e-4 relative (north_star);
      free running  every term inside the band the REFERENCE shows at this batch size under 1e-6 .. 1e-5 perturbations of its encoder
                    outputs (tests/golden/step_conditioning_bottle_b8x4.npz), encoder outputs within 1e-5 of the CPU's, poses 1e-4.
    Gradients of five probe parameters, both legs: relative L2 / cosine against the CPU oracle backend's."""
    import numpy as np
    import oracle_backend
    import bench
    import scp_amd.dino as dino
    from scp_amd import synthetic as synth
    dino.ALLOW_RANDOM_INIT = True
    bs, rep = 8, 4
    probes = {"mean_v": "mesh.mean_v", "resnet_conv1": "encoder.backbone.resnet.conv1.weight", "featnet_proj": "encoder.featnet.proj.weight",
              "pose_trans": "encoder.pose_predictor.trans_pred_layer.weight", "mesh_stn_fc": "encoder.featnet_mesh.stn.fc.weight"}

    def run(model, data):
        for p in model.parameters():
            p.grad = None
        model.iters = 0
        total, aux = model(data)
        total.mean().backward()
        params = dict(model.named_parameters())
        return ({k: float(v) for k, v in aux.items()}, [t.detach().cpu().double().numpy() for t in model.last_pose],
                {k: params[n].grad.detach().cpu().double().numpy().ravel() for k, n in probes.items()},
                tuple(t.detach().cpu() for t in model.last_geometry), tuple(t.detach().cpu() for t in model.last_features))

    def build(device):
        tr, _ = bench.build_trainer(device, 1, bs, rep)          # the bench's own builder: same seed, same options
        bench.pin_rng_consumers(tr.model)
        return tr.model

    with monkeypatch.context() as mp:
        oracle_backend.install(mp)
        cpu = build("cpu")
        ref_aux, ref_pose, ref_grad, ref_geo, ref_feat = run(cpu, synth.make_batch(bs, rep, 256, seed=100, device="cpu"))
        pc = cpu.pretrain_corr_net
        sel_nn, sel_topk = tuple(t.clone() for t in pc.last_nn), pc.last_topk.clone()
        del cpu
    from scp_amd.soft_renderer.cuda import soft_rasterize as native
    assert native.forward_soft_rasterize.__module__.startswith("scp_amd"), "HIP path must be the one that runs"
    data = synth.make_batch(bs, rep, 256, seed=100, device="cuda")
    band, _, _ = step_case.conditioning_band("step_conditioning_bottle_b8x4")
    report = {}
    for leg in ("free_running", "pinned"):
        gpu = build("cuda")
        gpu.pretrain_corr_net.nn_override = tuple(t.cuda() for t in sel_nn)
        gpu.pretrain_corr_net.topk_override = sel_topk.cuda()
        if leg == "pinned":
            bench.pin_encoder_outputs(gpu, ref_geo, ref_feat)
        got_aux, got_pose, got_grad, got_geo, _ = run(gpu, data)
        for k, ref in ref_aux.items():
            rel = abs(got_aux[k] - ref) / max(abs(ref), 1e-12)
            tol = 1e-4 if leg == "pinned" else band.get(k, 1e-4)
            print("%-12s %-22s cpu-oracle %.9g gpu %.9g rel %.2e (tol %.2e)" % (leg, k, ref, got_aux[k], rel, tol))
            report[(leg, k)] = (rel, tol)
        for k in probes:
            g, r = got_grad[k], ref_grad[k]
            rel = np.linalg.norm(g - r) / np.linalg.norm(r)
            cos = g @ r / (np.linalg.norm(g) * np.linalg.norm(r))
            print("%-12s grad %-14s rel L2 %.3e cos %.8f" % (leg, k, rel, cos))
            report[(leg, "grad_" + k)] = (rel, cos)
        if leg == "free_running":
            for name, a, b in zip(("pred_v", "rotation", "translation"), got_geo, ref_geo):
                d = float((a - b).abs().max())
                print("free_running encoder output %-12s max abs dev %.2e" % (name, d))
                assert d <= 1e-5, (name, d)
            np.testing.assert_allclose(got_pose[0], ref_pose[0], rtol=1e-4, atol=5e-5)
            np.testing.assert_allclose(got_pose[1], ref_pose[1], rtol=1e-4, atol=5e-5)
        del gpu
    bad = {k: v for k, v in report.items() if not k[1].startswith("grad_") and v[0] > v[1]}
    assert not bad, bad
    # gradients: the CPU side sums in other orders (oneDNN / C rasteriser in pixel order vs wavefront trees / atomics) and the ReLU /
    # hard-footprint branches of a few pixels flip with the encoder's rounding.  At this batch those effects average out; what is left
    # moves from run to run with the atomics' order (MI355X, round 5, four suite runs: pinned rel-L2 1.2e-3 ... 5.0e-3 on resnet conv1 --
    # the end of the longest backward chain -- <= 1e-3 elsewhere, cos >= 0.999987; free running <= 6.2e-3 / >= 0.999981) -- held to
    # 1.5e-2 / 0.9999 and 2e-2 / 0.9998 (the small-batch tests above keep their wider bands: there a single flipped pixel is a visible
    # share of a gradient)
    for (leg, k), (rel, cos) in report.items():
        if k.startswith("grad_"):
            lim_rel, lim_cos = (1.5e-2, 0.9999) if leg == "pinned" else (2e-2, 0.9998)
            assert rel <= lim_rel and cos >= lim_cos, (leg, k, rel, cos)


def test_trainer_step_runs_and_updates():
    import scp_amd.dino as dino
    from scp_amd.flags import Options
    from scp_amd.trainer import Trainer
    import scenes
    import synth
    dino.ALLOW_RANDOM_INIT = True
    opts = Options("laptop_wild6d", batch_size=2, repeat=2, train=True, total_iters=100)
    torch.manual_seed(0)
    tr = Trainer(opts, prior=scenes.bottle_like(3), device="cuda")
    data = synth.make_batch(2, 2, 256, seed=1, device="cuda")
    before = tr.model.encoder.featnet.proj.weight.detach().clone()
    losses = []
    for _ in range(3):
        total, aux, grad = tr.step(data)
        losses.append(float(total))
    assert all(l == l and abs(l) < 1e3 for l in losses)
    assert not torch.equal(before, tr.model.encoder.featnet.proj.weight)


def test_high_res_step_runs():
    """BASELINE configs[4] geometry in fp32: 512x512 images, corr_h = corr_w = 128 (ViT sequence 4097,
    16384 correspondence pixels), icosphere-4 mesh (2562 v / 5120 f): one full training step runs through
    every HIP kernel at those sizes and produces finite losses and gradients"""
    import scp_amd.dino as dino
    from scp_amd.flags import Options
    from scp_amd.trainer import Trainer
    import scenes
    import synth
    dino.ALLOW_RANDOM_INIT = True
    opts = Options("laptop_wild6d", batch_size=1, repeat=2, train=True, total_iters=100, img_size=512, corr_h=128,
                   corr_w=128)
    torch.manual_seed(0)
    tr = Trainer(opts, prior=scenes.bottle_like(4), device="cuda")
    data = synth.make_batch(1, 2, 512, seed=3, device="cuda")
    total, aux, grad = tr.step(data)
    assert torch.isfinite(total).all() and all(torch.isfinite(v).all() for v in aux.values())
    assert all(torch.isfinite(p.grad).all() for p in tr.model.parameters() if p.grad is not None)


@pytest.mark.parametrize("category", ["bottle", "bowl", "camera", "laptop", "mug"])
def test_every_wild6d_category_preset_steps(category):
    """BASELINE configs[4] names 'all 5 Wild6D categories': each shipped flag set (config/<cat>_wild6d/base_config.txt,
    restated in scp_amd.flags.PRESETS; symmetry_idx 0 = 17 rotations about y, 1 = mirror, -1 = none) runs two full
    training steps with finite losses and a real parameter update"""
    import scp_amd.dino as dino
    from scp_amd.flags import Options
    from scp_amd.trainer import Trainer
    import scenes
    import synth
    dino.ALLOW_RANDOM_INIT = True
    opts = Options(category + "_wild6d", batch_size=2, repeat=2, train=True, total_iters=100)
    torch.manual_seed(0)
    tr = Trainer(opts, prior=scenes.bottle_like(3), device="cuda")
    assert tr.model.mesh.symm_rots.shape[0] == {0: 17, 1: 2, -1: 1}[opts.symmetry_idx]
    data = synth.make_batch(2, 2, 256, seed=2, device="cuda")
    before = tr.model.mesh.mean_v.detach().clone()
    for _ in range(2):
        total, aux, grad = tr.step(data)
        assert torch.isfinite(total).all() and all(torch.isfinite(v).all() for v in aux.values())
    assert not torch.equal(before, tr.model.mesh.mean_v)


def test_lookahead_of_the_frozen_vit_changes_nothing_but_the_schedule(monkeypatch):
    """SCP_STREAMS=overlap (scp_amd/streams.py, the default schedule).
    Trainer.step(data, next_data): the DINO pass of the following batch is enqueued on the side stream before this step's
    backward (Trainer.train() and bench.py do that).  (1) What the look-ahead leaves for the next step -- features and pair
    matching of the NEXT batch, a different tensor than the current one -- is bit-identical to computing them when the step starts;
    (2) four steps on four different batches with and without it end in the same losses and parameters, up to the run-to-run
    spread of the step itself (atomics in the rasteriser's backward, amplified by the sigma = 1e-4 depth term and by training)."""
    import copy
    import scp_amd.dino as dino
    from scp_amd.flags import Options
    from scp_amd.trainer import Trainer
    import scenes
    import synth
    from scp_amd import streams
    monkeypatch.setattr(streams, "MODE", "overlap")
    dino.ALLOW_RANDOM_INIT = True
    batches = [synth.make_batch(2, 2, 256, seed=10 + i, device="cuda") for i in range(4)]
    runs, state = {}, None
    for look in (False, "again", True):
        opts = Options("laptop_wild6d", batch_size=2, repeat=2, train=True, total_iters=100)
        torch.manual_seed(0)
        tr = Trainer(opts, prior=scenes.bottle_like(3), device="cuda")
        if state is None:
            state = copy.deepcopy(tr.model.state_dict())
        tr.model.load_state_dict(state)
        tr.model.rotation_angle = 90.0
        torch.manual_seed(1)
        hist = []
        for i, data in enumerate(batches):
            nxt = batches[i + 1] if (look is True and i + 1 < len(batches)) else None
            total, aux, grad = tr.step(data, next_data=nxt)
            hist.append({k: float(v.detach()) for k, v in aux.items()})
            if nxt is not None and i == 1:
                # (1) the prefetched state for batch i + 1 against a synchronous evaluation of the same thing
                pc = tr.model.pretrain_corr_net
                img, feats, matched = pc._prefetched
                assert img is nxt[0]
                torch.cuda.synchronize()
                with torch.no_grad():
                    direct = pc.net.key_tokens(nxt[0], pc._keep_tokens(nxt[1]))
                    direct_matched = pc._match_pairs(direct, nxt[1])
                assert torch.equal(feats, direct)
                for u, v in zip(matched, direct_matched):
                    assert torch.equal(u, v)
        runs[look] = (hist, [p.detach().clone() for p in tr.model.parameters()])
    for a, b, c in zip(*[runs[k][0] for k in (False, "again", True)]):
        for k in a:
            floor = abs(a[k] - b[k])
            assert abs(c[k] - a[k]) <= 6 * floor + 5e-3 * abs(a[k]) + 1e-9, (k, a[k], b[k], c[k])
    for p, q, r in zip(runs[False][1], runs["again"][1], runs[True][1]):
        # `floor` is ONE sample of the run-to-run spread (float atomics in the rasteriser's backward; AdamW turns a gradient element
        # near zero into an update of +-lr whatever its size): 10 x floor, and never below a few AdamW steps at the initial lr (4e-6)
        floor = (p - q).abs().max().item()
        assert (r - p).abs().max().item() <= 10 * floor + 1e-3 * p.abs().max().item() + 1e-6


def test_mixed_bf16_step_tracks_fp32():
    """BASELINE configs[4] precision (opts.mixed_bf16: bf16 convolutions and ViT linears, fp32 everywhere else): the
    same model / batch in both precisions.  bf16 carries 8 mantissa bits, so this is a sanity band, not parity: every
    loss term within 5 % (or 2e-3 absolute) of its fp32 value, finite gradients."""
    import copy
    import scp_amd.dino as dino
    from scp_amd import imgops
    from scp_amd.flags import Options
    from scp_amd.trainer import Trainer
    import scenes
    import synth
    dino.ALLOW_RANDOM_INIT = True
    out = {}
    state = None
    for mixed in (False, True):
        opts = Options("laptop_wild6d", batch_size=2, repeat=2, train=True, total_iters=100, mixed_bf16=mixed)
        torch.manual_seed(0)
        tr = Trainer(opts, prior=scenes.bottle_like(3), device="cuda")
        if state is None:
            state = copy.deepcopy(tr.model.state_dict())
        tr.model.load_state_dict(state)
        tr.model.encoder.random_jitter = torch.nn.Identity()
        tr.model.rotation_angle = 90.0
        data = synth.make_batch(2, 2, 256, seed=4, device="cuda")
        torch.manual_seed(1)
        total, aux = tr.model(data)
        total.mean().backward()
        assert all(torch.isfinite(p.grad).all() for p in tr.model.parameters() if p.grad is not None)
        out[mixed] = {k: float(v.detach()) for k, v in aux.items()}
    dino.MIXED_BF16 = False
    for k, ref in out[False].items():
        if k == "cycle_loss_pretrain":
            continue            # discrete top-k / argmax selections on DINO features: re-selected under bf16
        assert abs(out[True][k] - ref) <= 5e-2 * abs(ref) + 2e-3, (k, out[True][k], ref)


def test_high_res_mixed_bf16_step_runs():
    """512x512, icosphere-4 mesh (2562 v / 5120 f), mixed bf16"""
    import scp_amd.dino as dino
    from scp_amd.flags import Options
    from scp_amd.trainer import Trainer
    import scenes
    import synth
    dino.ALLOW_RANDOM_INIT = True
    opts = Options("laptop_wild6d", batch_size=1, repeat=2, train=True, total_iters=100, img_size=512, corr_h=128,
                   corr_w=128, mixed_bf16=True)
    torch.manual_seed(0)
    tr = Trainer(opts, prior=scenes.bottle_like(4), device="cuda")
    data = synth.make_batch(1, 2, 512, seed=3, device="cuda")
    try:
        total, aux, grad = tr.step(data)
    finally:
        dino.MIXED_BF16 = False
    assert torch.isfinite(total).all() and all(torch.isfinite(v).all() for v in aux.values())


def test_training_reduces_the_loss_on_a_fixed_batch():
    """optimisation sanity on the full HIP path: 60 trainer steps on ONE fixed synthetic batch (jitter and rotation angle
    drawn fresh every step, as in training; OneCycle warm-up over the first 36) must lower the total loss and keep
    every step finite"""
    import scp_amd.dino as dino
    from scp_amd.flags import Options
    from scp_amd.trainer import Trainer
    import scenes
    import synth
    dino.ALLOW_RANDOM_INIT = True
    dino.MIXED_BF16 = False
    opts = Options("laptop_wild6d", batch_size=2, repeat=2, train=True, total_iters=120, learning_rate=3e-4)
    torch.manual_seed(0)
    tr = Trainer(opts, prior=scenes.bottle_like(3), device="cuda")
    data = synth.make_batch(2, 2, 256, seed=6, device="cuda")
    losses = []
    for _ in range(60):
        total, aux, grad = tr.step(data)
        losses.append(float(total.detach()))
    assert all(l == l and abs(l) < 1e4 for l in losses)
    first, last = sum(losses[:5]) / 5, sum(losses[-10:]) / 10
    assert last < 0.9 * first, (first, last, losses[::5])


def test_step_loop_does_not_stall_at_the_known_bad_stream_placements():
    """With three side streams the step loop had stream placements at which the device stopped, every stream waiting and no wavefront
    resident (profiles/r06_stall_rates_call4..10.txt); the default schedule, two side streams of the step's own and the texture pass on
    the main stream, did not stop at any of 14.  It must run through at three of those placements, with and without the multi-GPU
    schedule's communication stream (one-rank RCCL group).  One trial per fresh process (tests/step_trial.py), every wait bounded."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    script = os.path.join(root, "tests", "step_trial.py")

    def trial(pre, **env):
        e = dict(os.environ, SCP_DEVICE_TIMEOUT_S="10", **env)
        for k in ("SCP_SIDE_STREAMS", "SCP_FORCE_COLLECTIVES"):
            if k not in env:
                e.pop(k, None)
        r = subprocess.run([sys.executable, script, str(pre)], env=e, capture_output=True, text=True, timeout=150)
        lines = [l for l in r.stdout.splitlines() if l.startswith(("OK", "HANG"))]
        return lines[-1] if lines else "?? rc=%d %s" % (r.returncode, (r.stdout + r.stderr)[-400:])
    got = [trial(35), trial(3), trial(0), trial(35, SCP_FORCE_COLLECTIVES="1")]
    assert all(g.startswith("OK") for g in got), got
