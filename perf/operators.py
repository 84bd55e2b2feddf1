"""The operators around a tensor-parallel rank's decode step -- products with 4-bit weights, their
SwiGLU and rotary forms, the quantiser, and rotary positions on whole sequences -- as cases to
measure, each in a plain form made of elementary torch operations.

A 4-bit weight matrix [N, K] is codes 0..15, two per byte along K (the even column in the low half),
with one scale per row and group of `group` columns and, where it has them, one whole zero point
0..15 per row and group: w[n, k] = (code[n, k] - zero[n, k // group]) * scale[n, k // group].
Without zero points the zero is 8.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token through a small key/value projection: nothing but latency
        dict(name="token_1x1024x1024", op="gemm", M=1, N=1024, K=1024, group=64, zeros=False, dtype="bf16"),
        # one token through a rank's shard of a down projection
        dict(name="token_1x8192x3584", op="gemm", M=1, N=8192, K=3584, group=128, zeros=False, dtype="bf16"),
        # a few users' tokens, ragged everywhere, small groups with zero points
        dict(name="few_13x3581x8191", op="gemm", M=13, N=3581, K=8191, group=32, zeros=True, dtype="fp16"),
        # the decode batch of the GEMM+AllReduce benchmark
        dict(name="batch_128x8192x1024", op="gemm", M=128, N=8192, K=1024, group=128, zeros=True, dtype="bf16"),
        # one token through a rank's gate and up projections
        dict(name="mlp_token_1x7168x8192", op="swiglu", M=1, N=7168, K=8192, group=128, zeros=False, dtype="bf16"),
        # a chunk of a prompt, or 256 users, through whole gate and up projections
        dict(name="mlp_chunk_256x28672x8192", op="swiglu", M=256, N=28672, K=8192, group=64, zeros=True, dtype="bf16"),
        # four users' tokens through a rank's shard of a query/key/value projection, far into a context
        dict(name="qkv_4x10x128x8192", op="qkv", M=4, K=8192, heads=10, rotated=9, head_dim=128, rotary_dim=128,
             interleaved=False, group=128, zeros=False, dtype="bf16", far=1000000),
        # a batch through a whole projection whose heads are turned in part, in pairs of neighbours
        dict(name="qkv_96x48x96x4096", op="qkv", M=96, K=4096, heads=48, rotated=40, head_dim=96, rotary_dim=32,
             interleaved=True, group=32, zeros=True, dtype="fp16", far=32768),
        # weights quantised when a model is loaded, and read back
        dict(name="quantize_8192x8192", op="quantize", N=8192, K=8192, group=128, zeros=False, dtype="bf16"),
        # the same for an adapter's odd matrix
        dict(name="quantize_1025x999", op="quantize", N=1025, K=999, group=32, zeros=True, dtype="fp16"),
        # the queries and keys of a prompt
        dict(name="rotary_8192x40x128", op="rotary", T=8192, heads=40, head_dim=128, rotary_dim=128, interleaved=False,
             inverse=False, dtype="bf16", far=8192),
        # the gradient of a partly turned head, odd sizes, scaled for a long context
        dict(name="rotary_back_4097x9x80", op="rotary", T=4097, heads=9, head_dim=80, rotary_dim=40, interleaved=True,
             inverse=True, dtype="fp32", far=1000000),
    ]


def _size(rng, lo, hi):
    """A size between lo and hi, even over the logarithm; half of them round, half as they come."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and n >= 64:
        n = n // 32 * 32
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "swiglu", "qkv", "quantize", "rotary"])
    kind = dict(group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16"]))
    if op in ("gemm", "swiglu"):
        M, N, K = _size(rng, 1, 256), _size(rng, 64, 28672), _size(rng, 64, 28672)
        while N * K > 28672 * 8192:
            N, K = max(64, N // 2), K // 2 + 1
        return dict(op=op, M=M, N=N + N % 2 if op == "swiglu" else N, K=K, **kind)
    if op == "qkv":
        head_dim = rng.choice([64, 80, 96, 128, 256])
        heads = rng.randint(3, 60)
        return dict(op=op, M=_size(rng, 1, 256), K=_size(rng, 64, 8192), heads=heads, rotated=rng.randint(1, heads),
                    head_dim=head_dim, rotary_dim=rng.choice([head_dim, head_dim // 2, 16]),
                    interleaved=rng.random() < 0.5, far=rng.choice([4096, 131072, 1000000]), **kind)
    if op == "quantize":
        return dict(op=op, N=_size(rng, 1, 8192), K=_size(rng, 1, 8192), **kind)
    head_dim = rng.choice([64, 80, 96, 128, 256])
    heads = rng.randint(1, 64)
    return dict(op=op, T=_size(rng, 1, max(1, 8192 * 40 * 128 // (heads * head_dim * 2))), heads=heads, head_dim=head_dim,
                rotary_dim=rng.choice([head_dim, head_dim // 2, 16]), interleaved=rng.random() < 0.5,
                inverse=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                far=rng.choice([4096, 131072, 1000000]))


# ------------------------------------------------------------------------------------- inputs
def _divisor(s):
    """A scale of nothing (a group of zeros) divides as one: every code of the group then means zero."""
    return torch.where(s == 0, torch.ones_like(s), s)


def _make_codes(w, group, zeros, dtype):
    """Codes, scales and zero points of a checkpoint for the weights w [N, K] (fp32)."""
    N, K = w.shape
    G = -(-K // group)
    w = torch.nn.functional.pad(w, (0, G * group - K)).view(N, G, group)
    if zeros:
        lo, hi = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        s = ((hi - lo) / 15).to(dtype)
        z = (-lo / _divisor(s.float())).round().clamp(0, 15)
    else:
        s = (w.abs().amax(-1) / 7).to(dtype)
        z = torch.full((N, G), 8.0, device=w.device)
    q = (w.div_(_divisor(s.float()).unsqueeze(-1)).round_().add_(z.unsqueeze(-1))).clamp_(0, 15).to(torch.uint8)
    q = q.view(N, G * group)
    q[:, K:] = 0
    q = q[:, :K + K % 2]
    return q[:, 0::2] | (q[:, 1::2] << 4), s, z.to(torch.uint8) if zeros else None


def _frequencies(rotary_dim, far):
    """Radians per position of each pair, interpolated by parts where the context is a long one."""
    f = 500000.0 ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    if far > 8192:
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1) / 3).clamp(0, 1)
        f = f * keep + f / 8 * (1 - keep)
    return f.float().cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    st = dict(case=case, dtype=dtype)
    if op == "rotary":
        st["x"] = torch.randn((case["T"], case["heads"], case["head_dim"]), device="cuda", generator=g).to(dtype)
        st["y"] = torch.empty_like(st["x"])
    elif op == "quantize":
        w = torch.randn((case["N"], case["K"]), device="cuda", generator=g)
        st["w"] = (w * 0.02).to(dtype)
        st["y"] = torch.empty_like(st["w"])
    else:
        M, K = case["M"], case["K"]
        N = case["heads"] * case["head_dim"] if op == "qkv" else case["N"]
        w = torch.randn((N, K), device="cuda", generator=g).mul_(K ** -0.5)
        st["codes"], st["scales"], st["zeros"] = _make_codes(w, case["group"], case["zeros"], dtype)
        del w
        # activations: normal, with a few channels far louder than the others
        loud = torch.rand((1, K), device="cuda", generator=g) < 0.01
        st["x"] = (torch.randn((M, K), device="cuda", generator=g) * torch.where(loud, 8.0, 1.0)).to(dtype)
        st["y"] = torch.empty((M, N // 2 if op == "swiglu" else N), device="cuda", dtype=dtype)
        if own:
            from mkernel_b200 import ops
            form = {}
            if op == "swiglu":
                form = dict(form="gate_up")
            elif op == "qkv":
                form = dict(form="rotary", head_dim=case["head_dim"], rotary_dim=case["rotary_dim"],
                            rotated_heads=case["rotated"], interleaved=case["interleaved"])
            # laid out once, when a program loads its weights
            st["weight"] = ops.w4_pack(st["codes"], st["scales"], st["zeros"], K=K, **form)
    if "far" in case:
        rows = case["T"] if op == "rotary" else case["M"]
        st["freq"] = _frequencies(case["rotary_dim"], case["far"])
        first = torch.randint(0, max(1, case["far"] - rows), (1,), device="cuda", generator=g)
        if op == "rotary":                 # one sequence, row after row
            st["pos"] = first + torch.arange(rows, device="cuda")
        else:                              # users, each at a position of its own
            st["pos"] = torch.randint(0, case["far"], (rows,), device="cuda", generator=g)
        st["scale"] = 1.0 if case["far"] <= 8192 else 0.1 * math.log(8.0) + 1.0
    return st


# ------------------------------------------------------------------------------------- one pass
def _weights(st):
    """The 4-bit weights as fp32 [N, K]."""
    K, group = st["case"]["K"], st["case"]["group"]
    q = torch.stack((st["codes"] & 15, st["codes"] >> 4), dim=-1).view(st["codes"].shape[0], -1)[:, :K].float()
    z = 8.0 if st["zeros"] is None else st["zeros"].float().repeat_interleave(group, 1)[:, :K]
    return (q - z) * st["scales"].float().repeat_interleave(group, 1)[:, :K]


def _turn(x, pos, freq, scale, interleaved, inverse=False):
    """x [T, heads, D] in fp32: the first 2 * len(freq) features of every head turned."""
    r = 2 * freq.numel()
    angle = pos.double().view(-1, 1) * freq.double()
    if inverse:
        angle = -angle
    cos, sin = (torch.cos(angle) * scale).float().unsqueeze(1), (torch.sin(angle) * scale).float().unsqueeze(1)
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, v), dim=-1).flatten(-2) if interleaved else torch.cat((u, v), dim=-1)
    return torch.cat((turned, x[..., r:]), dim=-1)


def run(st):
    c, op = st["case"], st["case"]["op"]
    if own:
        from mkernel_b200 import ops
        if op == "gemm":
            ops.w4_gemm(st["x"], st["weight"], st["y"])
        elif op == "swiglu":
            ops.w4_gemm_swiglu(st["x"], st["weight"], st["y"])
        elif op == "qkv":
            ops.w4_gemm_rotary(st["x"], st["weight"], st["y"], st["pos"], st["freq"], scale=st["scale"])
        elif op == "quantize":
            ops.w4_quantize(st["w"], group=c["group"], zero_points=c["zeros"]).dequantize(st["y"])
        else:
            ops.rotary(st["x"], st["pos"], st["freq"], st["y"], interleaved=c["interleaved"], inverse=c["inverse"],
                       scale=st["scale"])
        return st["y"]
    if op == "rotary":
        y = _turn(st["x"].float(), st["pos"], st["freq"], st["scale"], c["interleaved"], c["inverse"])
        return y.to(st["dtype"])
    if op == "quantize":
        w, (N, K), group = st["w"].float(), st["w"].shape, c["group"]
        G = -(-K // group)
        w = torch.nn.functional.pad(w, (0, G * group - K)).view(N, G, group)
        if c["zeros"]:
            lo, hi = w.amin(-1, keepdim=True).clamp(max=0), w.amax(-1, keepdim=True).clamp(min=0)
            s = ((hi - lo) / 15).to(st["dtype"]).float()
            z = (-lo / _divisor(s)).round().clamp(0, 15)
            q = ((w / _divisor(s)).round() + z).clamp(0, 15) - z
        else:
            s = (w.abs().amax(-1, keepdim=True) / 7).to(st["dtype"]).float()
            q = (w / _divisor(s)).round().clamp(-8, 7)
        return (q * s).view(N, G * group)[:, :K].to(st["dtype"]).contiguous()
    y = torch.matmul(st["x"].float(), _weights(st).t())
    if op == "swiglu":
        gate, up = y.chunk(2, dim=1)
        y = gate / (1 + torch.exp(-gate)) * up
    elif op == "qkv":
        y = y.view(c["M"], c["heads"], c["head_dim"])
        turned = _turn(y[:, :c["rotated"]], st["pos"], st["freq"], st["scale"], c["interleaved"])
        y = torch.cat((turned, y[:, c["rotated"]:]), dim=1).view(c["M"], -1)
    return y.to(st["dtype"])


# ------------------------------------------------------------------------------------- work, exact
def work(case):
    op = case["op"]
    if op == "rotary":
        n = case["T"] * case["heads"] * case["head_dim"]
        return {"bytes": 2 * n * (4 if case["dtype"] == "fp32" else 2) + 8 * case["T"], "flops": 3 * n}
    N = case["heads"] * case["head_dim"] if op == "qkv" else case["N"]
    groups = N * -(-case["K"] // case["group"])
    held = N * case["K"] / 2 + groups * (2.5 if case["zeros"] else 2)
    if op == "quantize":
        return {"bytes": 4 * N * case["K"] + held, "flops": 6 * N * case["K"]}
    M = case["M"]
    return {"bytes": held + 2 * M * case["K"] + 2 * M * (N // 2 if op == "swiglu" else N), "flops": 2 * M * N * case["K"]}


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]

    def turned(y, sign):
        D, r = case["head_dim"], case["rotary_dim"]
        phase = sign * st["pos"].to(torch.float64)[:, None] * st["freq"].to(torch.float64)[None, :]
        w = torch.polar(torch.full_like(phase, st["scale"]), phase)[:, None, :]
        out = y.clone()
        first = torch.arange(r // 2, device=y.device) * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else r // 2)
        z = torch.complex(y[..., first], y[..., second]) * w
        out[..., first], out[..., second] = z.real, z.imag
        return out

    if op == "rotary":
        return turned(st["x"].double(), -1.0 if case["inverse"] else 1.0)
    if op == "quantize":
        # Codes are whole numbers chosen by comparisons of values of the inputs' type: which code is the
        # nearest follows the scale as it is held, so 64 bits change nothing but the last product.
        w, group = st["w"].double(), case["group"]
        N, K = w.shape
        out = torch.empty_like(w)
        for k in range(0, K, group):
            part = w[:, k:k + group]
            if case["zeros"]:
                lo, hi = part.amin(1).clamp(max=0), part.amax(1).clamp(min=0)
                s = ((hi - lo).float() / 15).to(st["dtype"]).double()[:, None]
                z = torch.round(-lo[:, None] / s).nan_to_num(0.0).clamp(0, 15)
                out[:, k:k + group] = s * ((torch.round(part / s).nan_to_num(0.0) + z).clamp(0, 15) - z)
            else:
                s = (part.abs().amax(1).float() / 7).to(st["dtype"]).double()[:, None]
                out[:, k:k + group] = s * torch.round(part / s).nan_to_num(0.0).clamp(-8, 7)
        return out
    K, group = case["K"], case["group"]
    cols = torch.arange(K, device="cuda")
    x = st["x"].double()
    rows = []
    for n in range(0, st["codes"].shape[0], 4096):
        codes = st["codes"][n:n + 4096]
        nib = (codes[:, cols // 2] >> (4 * (cols % 2)).to(torch.uint8)) & 15
        w = nib.double()
        w -= 8 if st["zeros"] is None else st["zeros"][n:n + 4096].double()[:, cols // group]
        w *= st["scales"][n:n + 4096].double()[:, cols // group]
        rows.append(torch.einsum("nk,mk->mn", w, x))
    y = torch.cat(rows, dim=1)
    if op == "swiglu":
        half = y.shape[1] // 2
        return torch.special.expit(y[:, :half]) * y[:, :half] * y[:, half:]
    if op == "qkv":
        y = y.view(case["M"], case["heads"], case["head_dim"])
        y = torch.cat((turned(y[:, :case["rotated"]], 1.0), y[:, case["rotated"]:]), dim=1).view(case["M"], -1)
    return y
