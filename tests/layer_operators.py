"""A small DiT run with every option of the layer at once -- rotary positions on three axes, a sliding window with the
prompt visible, adapters on the four projections -- and the same model in plain torch. Used by the CPU and GPU tests."""
import math
import os
import socket
import sys

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
PKG = os.path.join(ROOT, "minimaxh3-on-a100-x4_b200")
CFG = dict(n_blocks=2, hidden=512, heads=8, head_dim=128, ffn=1024, t_dim=64)


def free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def setup(S, dev):
    import h3_model as M
    import h3attn as O
    model = M.MiniMaxH3Model(**CFG, dtype=torch.bfloat16, device=dev)
    M.init_weights(model, 21, std=0.03)
    for blk in model.blocks:  # open gates: attention and FFN weigh as much as the residual stream
        bias = blk.adaln_proj.lin.bias.data.view(6, -1)
        bias[2], bias[5] = 1.0, 1.0
    g = torch.Generator().manual_seed(S)
    h = torch.randn(S, CFG["hidden"], generator=g).to(torch.bfloat16).to(dev)
    t_emb = M.timestep_embedding(torch.tensor([500.0, 250.0]), CFG["t_dim"]).to(torch.bfloat16).to(dev)
    segs = [(0, 50, 0), (50, S, 1)]
    i = torch.arange(S)
    pos = torch.stack([i // 48, (i // 8) % 6, i % 8], 1).int().to(dev)
    rope = O.RopePositions(pos, *O.rope_axes_freqs([16, 24, 24], device=dev))
    stacks = []
    for blk in model.blocks:
        for lin in (blk.attn.qkv_proj, blk.attn.out_proj, blk.mlp.fc1, blk.mlp.fc2):
            n, k = lin.weight.shape
            pairs = [((torch.randn(r, k, generator=g) * k ** -0.5).to(torch.bfloat16).to(dev),
                      (torch.randn(n, r, generator=g) * 0.2).to(torch.bfloat16).to(dev)) for r in (4, 16, 9)]
            stacks.append((lin, O.stack_adapters(pairs, [0.5, 1.0, -0.7])))
    options = {"h3_window": {"left": 60, "right": 20, "sinks": 30},
               "h3_adapter_segments": [(0, 40, 2), (40, S // 2, 0), (S // 2 + 30, S, 1)]}
    return model, h, t_emb, segs, rope, stacks, options


def plain(model, h, t_emb, segs, rope, stacks, options):
    """The block loop in fp32 torch ops (weights as they are)."""
    import h3_model as M
    S, dev = h.shape[0], h.device
    ad = {lin: s for lin, s in stacks}
    rows = torch.full((S,), -1, device=dev)
    for a, b, g in options.get("h3_adapter_segments", ()):
        rows[a:b] = g
    axis = rope.axis.long()
    ang = rope.pos.double()[:, axis.clamp_min(0)] * rope.inv_freq * (axis >= 0)
    c, s = ang.cos(), ang.sin()
    table = torch.stack([torch.stack([c, -s], -1), torch.stack([s, c], -1)], -2).float()
    p, j = torch.arange(S, device=dev)[:, None], torch.arange(S, device=dev)[None]
    w = options.get("h3_window")
    see = torch.ones(S, S, dtype=torch.bool, device=dev)
    if w is not None:
        see = ((j >= p - w["left"]) & (j <= p + w["right"])) | (j < w["sinks"])

    def lin(x, mod):
        y = x @ mod.weight.float().T
        if mod in ad and options.get("h3_adapter_segments"):
            a, b, scale = ad[mod]
            r = a.shape[0] // len(scale)
            mine = rows[:, None] == torch.arange(a.shape[0], device=dev)[None] // r
            y = y + (x @ a.float().T * mine * scale.repeat_interleave(r)) @ b.float().T
        return y

    x = h.float()
    H, D = CFG["heads"], CFG["head_dim"]
    ln = torch.nn.functional.layer_norm
    for blk in model.blocks:
        m = (torch.nn.functional.silu(t_emb.float()) @ blk.adaln_proj.lin.weight.float().T +
             blk.adaln_proj.lin.bias.float()).chunk(6, dim=-1)
        y = M._mod_scale_shift(ln(x, (x.shape[1],), eps=1e-6), m[0], m[1], segs)
        q, k, v = (t.reshape(S, H, D) for t in lin(y, blk.attn.qkv_proj).split(H * D, -1))
        q, k = (M.rms_rope_ref(t, n.weight, table, 1e-6).transpose(0, 1)
                for t, n in ((q, blk.attn.q_norm), (k, blk.attn.k_norm)))
        sc = (q @ k.transpose(1, 2) / math.sqrt(D)).masked_fill(~see, -math.inf)
        o = (torch.softmax(sc, -1) @ v.transpose(0, 1)).transpose(0, 1).reshape(S, H * D)
        x = M._mod_gate(x, m[2], lin(o, blk.attn.out_proj), segs)
        y = M._mod_scale_shift(ln(x, (x.shape[1],), eps=1e-6), m[3], m[4], segs)
        a, b = lin(y, blk.mlp.fc1).chunk(2, -1)
        x = M._mod_gate(x, m[5], lin(torch.nn.functional.silu(a) * b, blk.mlp.fc2), segs)
    return x


def worker(rank, world, port, S, out_dir, overlap, on_gpu):
    for p in (PKG, ROOT, HERE):
        if p not in sys.path:
            sys.path.insert(0, p)
    os.environ.update(RANK=str(rank), WORLD_SIZE=str(world), MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port),
                      LOCAL_RANK=str(rank))
    if not on_gpu:
        os.environ["SP_BACKEND"] = "gloo"
    if overlap:
        os.environ["SP_OVERLAP"] = overlap
    import h3_model as M
    import sp_runtime
    if not on_gpu:
        from oracle import cpu_ops
        sp_runtime._ops = cpu_ops
    sp_runtime.init(timeout_s=120)
    dev = torch.device("cuda", torch.cuda.current_device()) if on_gpu else torch.device("cpu")
    try:
        model, h, t_emb, segs, rope, stacks, options = setup(S, dev)
        sp_runtime.install(M)
        run = lambda opt: M.MiniMaxH3Model.run_blocks(model, h.clone(), t_emb, segs, rope, opt).float().cpu()  # noqa: E731
        with torch.no_grad():
            bare = run({"h3_window": options["h3_window"]})
            for lin, stack in stacks:
                sp_runtime.set_adapters(lin, stack)
            out = run(options)
            unnamed = run({"h3_window": options["h3_window"]})  # adapters attached, no segments: the bare model
            dense = run({"h3_adapter_segments": options["h3_adapter_segments"]})
            for lin, _ in stacks:
                sp_runtime.set_adapters(lin, None)
            off = run(options)
        if rank == 0:
            torch.save({"out": out, "bare": bare, "unnamed": unnamed, "dense": dense, "off": off},
                       os.path.join(out_dir, f"w{world}.pt"))
            if world == 1:
                opt = dict(options)
                opt.pop("h3_window")
                with torch.no_grad():
                    torch.save({"out": plain(model, h, t_emb, segs, rope, stacks, options).cpu(),
                                "dense": plain(model, h, t_emb, segs, rope, stacks, opt).cpu()},
                               os.path.join(out_dir, "plain.pt"))
    finally:
        if torch.distributed.is_initialized():
            torch.distributed.barrier()
            torch.distributed.destroy_process_group()


def run(world, S, out_dir, overlap=None, on_gpu=False):
    import torch.multiprocessing as mp
    mp.start_processes(worker, args=(world, free_port(), S, str(out_dir), overlap, on_gpu), nprocs=world,
                       start_method="spawn")
    return torch.load(os.path.join(out_dir, f"w{world}.pt"))


def near(a, b):
    """Two bf16 runs of the same blocks, or one and the fp32 model: every op rounds to bf16 (2^-8) some ten times a
    block, so the mean difference stays well below 2 % of the mean magnitude."""
    return (a - b).abs().mean().item() < 2e-2 * b.abs().mean().item()


# A bf16 run against the fp32 model, row by row: every op of a block rounds to bf16, ten roundings in a row of them,
# each off by at most 2^-8 of a value and by 2^-8 / sqrt(3) in the root mean square over a row. Two blocks, all errors
# added at their full size: 20 * 2^-8 / sqrt(3) = 4.5 % of the row's length.
ROW_BOUND = 20 * 2 ** -8 / math.sqrt(3)


def row_errors(a, b):
    """Relative L2 error of each token's row of a against b's."""
    return (a - b).norm(dim=1) / b.norm(dim=1)


def mistakes(S):
    """Options that differ from setup(S)'s at a single token or key: segments and window edges one off."""
    model, h, t_emb, segs, rope, stacks, options = setup(S, torch.device("cpu"))
    w, (first, second, third) = options["h3_window"], options["h3_adapter_segments"]
    changes = [{"h3_adapter_segments": s} for s in (
        [(0, first[1] + 1, 2), (first[1] + 1, second[1], 0), third], [first, (40, second[1] - 1, 0), third],
        [first, second, (third[0] + 1, S, 1)], [first, second, (third[0], S - 1, 1)])]
    changes += [{"h3_window": dict(w, **{k: w[k] + d})} for k, d in (("sinks", -1), ("left", 1), ("right", 1))]
    for change in changes:
        with torch.no_grad():
            yield change, plain(model, h, t_emb, segs, rope, stacks, dict(options, **change))
