"""The 8-bit operators of the framework as cases that can be timed and compared.

Four operators: the matrix product of e4m3 operands with a scale for each block of 128 ("linear"), the same with the
gated unit and the next product's quantisation on its way out ("gated"), the norms behind a part and in front of the
next one with a gate and a residual factor between them ("norms"), and the quantisation of rows and of weight blocks
("quantize").

Every quantised matrix is a pair (values e4m3, scales float32): for a group of 128 neighbouring elements of a row, or a
block of 128 x 128 elements of a weight, with a its largest magnitude, s = max(a / 448, 2^-126) and q = e4m3(x * (1 / s)).

``own`` false: the operators in elementary torch operations in 32 bits.  ``own`` true: the framework's kernels.
"""

import math

import torch

own = False

FP8 = torch.float8_e4m3fn
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
TINY = 2.0 ** -126


def listed():
    return [
        # a decoded token's attention output projection at the layer sizes of an 8B model: latency and the weight's bytes
        {"name": "linear, 1 token", "op": "linear", "T": 1, "N": 4096, "K": 4096, "out": "bfloat16"},
        # the down projection of a 14B model for a decode batch of no round number
        {"name": "linear, 61 tokens", "op": "linear", "T": 61, "N": 5120, "K": 17408, "out": "bfloat16"},
        # sizes that no tile divides, a last group of 80 elements, a float32 run
        {"name": "linear, ragged", "op": "linear", "T": 300, "N": 1000, "K": 1104, "out": "float32"},
        # a prompt chunk through the stacked q, k, v projection of a 14B model
        {"name": "linear, 1024 tokens", "op": "linear", "T": 1024, "N": 7168, "K": 5120, "out": "bfloat16"},
        # a long prompt's step through the down projection of an 8B model
        {"name": "linear, 4096 tokens", "op": "linear", "T": 4096, "N": 4096, "K": 12288, "out": "bfloat16"},
        # a decode batch of 8 through gate and up of an 8B model
        {"name": "gated, 8 tokens", "op": "gated", "T": 8, "I": 12288, "K": 4096},
        # decode beside a short prompt portion, 14B
        {"name": "gated, 100 tokens", "op": "gated", "T": 100, "I": 17408, "K": 5120},
        # a prompt of 2048 tokens, 8B
        {"name": "gated, 2048 tokens", "op": "gated", "T": 2048, "I": 12288, "K": 4096},
        # between two parts of a decode step: no norm behind, a bfloat16 stream, what the next product reads
        {"name": "norms, 8 tokens", "op": "norms", "T": 8, "H": 4096, "stream": "bfloat16", "delta": "bfloat16", "post": False,
         "gate": "none", "out": "fp8"},
        # between two parts of a long prompt's step: norms on both sides, a gate for every token, a float32 stream
        {"name": "norms, 4096 tokens", "op": "norms", "T": 4096, "H": 5120, "stream": "float32", "delta": "bfloat16", "post": True,
         "gate": "rows", "out": "bfloat16"},
        # the attention's output of a long prompt's step on its way into the output projection
        {"name": "quantize, rows", "op": "quantize", "T": 4096, "K": 8192, "dtype": "bfloat16", "block": 1},
        # a weight of an 8B model as it is loaded
        {"name": "quantize, blocks", "op": "quantize", "T": 12288, "K": 4096, "dtype": "bfloat16", "block": 128},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "gated", "norms", "quantize"))
    if op in ("linear", "gated"):
        while True:
            T, N, K = _log(rng, 1, 8192), _log(rng, 64, 16384), 16 * _log(rng, 4, 1024)
            if T * N * K * (2 if op == "gated" else 1) <= 1 << 37 and N * K <= 1 << 26:
                break
        if op == "linear":
            return {"op": op, "T": T, "N": N, "K": K, "out": rng.choice(("bfloat16", "float32"))}
        return {"op": op, "T": T, "I": N, "K": K}
    T, H = _log(rng, 1, 8192), _log(rng, 96, 12288)
    if rng.random() < 0.5:
        H = (H + 127) // 128 * 128          # what most models have
    while T * H > 5120 * 4096:
        T = T // 2 + 1
    if op == "norms":
        return {"op": op, "T": T, "H": H, "stream": rng.choice(("bfloat16", "float32")), "delta": rng.choice(("bfloat16", "float32")),
                "post": rng.random() < 0.7, "gate": rng.choice(("none", "channels", "rows")), "out": rng.choice(("fp8", "bfloat16", "float32"))}
    return {"op": op, "T": T, "K": H, "dtype": rng.choice(("bfloat16", "float32")), "block": rng.choice((1, 128))}


def _groups(n):
    return (n + 127) // 128


def _empty_rows(T, K, device="cuda"):
    """An e4m3 matrix with rows of a multiple of 16 bytes, and its scales."""
    return (torch.empty((T, (K + 15) // 16 * 16), dtype=FP8, device=device)[:, :K],
            torch.empty((T, _groups(K)), dtype=torch.float32, device=device))


def _spread(scales, rows, columns, block):
    """The scales, one for every element they stand for."""
    s = scales.repeat_interleave(128, 1)[:, :columns]
    return s if block == 1 else s.repeat_interleave(128, 0)[:rows]


def _amax(x, block):
    """The largest magnitude of every group (block 1) or block of 128 x 128 (block 128)."""
    T, K = x.shape
    G = _groups(K)
    a = torch.nn.functional.pad(x.abs(), (0, G * 128 - K)).view(T, G, 128).amax(2)
    if block == 1:
        return a
    R = _groups(T)
    return torch.nn.functional.pad(a, (0, 0, 0, R * 128 - T)).view(R, 128, G).amax(1)


def _quantized(x, block):
    """(values e4m3, scales) of the float matrix x."""
    s = (_amax(x, block) / 448.0).clamp_min(TINY)
    return (x * _spread(1.0 / s, *x.shape, block)).to(FP8), s


def _weight(N, K, gen):
    """A quantised weight [N, K]: normal with a deviation of 0.02, some input channels larger than others."""
    w = torch.empty((N, K), device="cuda").normal_(0.0, 0.02, generator=gen)
    w *= torch.empty(K, device="cuda").uniform_(0.5, 1.5, generator=gen)
    q, s = _quantized(w, 128)
    kept, _ = _empty_rows(N, K)
    kept.view(torch.uint8).copy_(q.view(torch.uint8))
    return kept, s


def _activations(T, K, gen):
    """Rows as a norm leaves them: normal, a few channels that stand out, tokens of different size."""
    x = torch.empty((T, K), device="cuda").normal_(generator=gen)
    x *= torch.empty((T, 1), device="cuda").uniform_(0.5, 2.0, generator=gen)
    x[:, torch.randint(0, K, (max(1, K // 256),), device="cuda", generator=gen)] *= 12.0
    return x


def _activations_quantized(T, K, gen):
    q, s = _quantized(_activations(T, K, gen), 1)
    kept, _ = _empty_rows(T, K)
    kept.view(torch.uint8).copy_(q.view(torch.uint8))
    return kept, s


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, T = case["op"], case["T"]
    state = dict(case)
    if op == "linear":
        state["x"], state["x_scales"] = _activations_quantized(T, case["K"], gen)
        state["w"], state["w_scales"] = _weight(case["N"], case["K"], gen)
        state["y"] = torch.empty((T, case["N"]), dtype=TYPES[case["out"]], device="cuda")
    elif op == "gated":
        state["x"], state["x_scales"] = _activations_quantized(T, case["K"], gen)
        state["gate"], state["gate_scales"] = _weight(case["I"], case["K"], gen)
        state["up"], state["up_scales"] = _weight(case["I"], case["K"], gen)
        state["y"], state["y_scales"] = _empty_rows(T, case["I"])
    elif op == "norms":
        H = case["H"]
        state["x"] = (3.0 * _activations(T, H, gen)).to(TYPES[case["stream"]])
        state["d"] = (0.3 * _activations(T, H, gen)).to(TYPES[case["delta"]])
        state["post_weight"] = torch.empty(H, device="cuda").normal_(1.0, 0.1, generator=gen) if case["post"] else None
        state["weight"] = torch.empty(H, device="cuda").normal_(1.0, 0.1, generator=gen)
        shape = {"none": None, "channels": (H,), "rows": (T, H)}[case["gate"]]
        state["g"] = None
        if shape is not None:
            state["g"] = torch.empty(shape, device="cuda").normal_(0.6, 0.3, generator=gen)
            if case["gate"] == "rows":
                state["g"] = state["g"].to(TYPES[case["delta"]])
        state["c"] = 0.75 if case["gate"] != "none" else 1.0
        if case["out"] == "fp8":
            state["y"], state["y_scales"] = _empty_rows(T, H)
        else:
            state["y"], state["y_scales"] = torch.empty((T, H), dtype=TYPES[case["out"]], device="cuda"), None
    else:
        x = _activations(T, case["K"], gen)
        state["x"] = (x * (0.02 if case["block"] == 128 else 1.0)).to(TYPES[case["dtype"]])
        state["y"], state["y_scales"] = _empty_rows(T, case["K"])
        if case["block"] == 128:
            state["y_scales"] = torch.empty((_groups(T), _groups(case["K"])), dtype=torch.float32, device="cuda")
    return state


def _run_own(st):
    from acvram_b200.kernels import ops
    op = st["op"]
    if op == "linear":
        return ops.linear_fp8(st["x"], st["x_scales"], st["w"], st["w_scales"], st["y"])
    if op == "gated":
        return ops.linear_fp8_swiglu(st["x"], st["x_scales"], st["gate"], st["gate_scales"], st["up"], st["up_scales"],
                                     st["y"], st["y_scales"])
    if op == "norms":
        ops.add_gated_norms(st["x"], st["d"], st["y"], st["y_scales"], post_weight=st["post_weight"], post_eps=1e-6, gate=st["g"],
                            residual_scale=st["c"], weight=st["weight"], eps=1e-6)
        return [st["x"], st["y"]] if st["y_scales"] is None else [st["x"], st["y"], st["y_scales"]]
    return ops.quantize_fp8(st["x"], st["y"], st["y_scales"], block_rows=st["block"])


def _product(x, x_scales, w, w_scales):
    return (x.float() * _spread(x_scales, *x.shape, 1)) @ (w.float() * _spread(w_scales, *w.shape, 128)).t()


def run(state):
    if own:
        return _run_own(state)
    op = state["op"]
    if op == "linear":
        return _product(state["x"], state["x_scales"], state["w"], state["w_scales"]).to(state["y"].dtype)
    if op == "gated":
        g = _product(state["x"], state["x_scales"], state["gate"], state["gate_scales"])
        u = _product(state["x"], state["x_scales"], state["up"], state["up_scales"])
        return _quantized(g / (1.0 + torch.exp(-g)) * u, 1)
    if op == "norms":
        x = state["x"]
        d = state["d"].float()
        if state["post_weight"] is not None:
            d = d / torch.sqrt(d.square().mean(1, keepdim=True) + 1e-6) * state["post_weight"]
        if state["g"] is not None:
            d = d * state["g"].float()
        x.copy_(x.float() + state["c"] * d)         # the stream is kept, in its own type
        kept = x.float()
        h = kept / torch.sqrt(kept.square().mean(1, keepdim=True) + 1e-6) * state["weight"]
        if state["y_scales"] is None:
            return [x, h.to(state["y"].dtype)]
        return [x, *_quantized(h, 1)]
    return _quantized(state["x"].float(), state["block"])


def work(case):
    op, T = case["op"], case["T"]
    if op == "linear":
        N, K = case["N"], case["K"]
        G = _groups(K)
        return {"bytes": T * K + 4 * T * G + N * K + 4 * _groups(N) * G + T * N * TYPES[case["out"]].itemsize, "flops": 2 * T * N * K}
    if op == "gated":
        I, K = case["I"], case["K"]
        G = _groups(K)
        return {"bytes": T * K + 4 * T * G + 2 * (I * K + 4 * _groups(I) * G) + T * I + 4 * T * _groups(I), "flops": 4 * T * I * K}
    if op == "norms":
        H = case["H"]
        out = T * H + 4 * T * _groups(H) if case["out"] == "fp8" else T * H * TYPES[case["out"]].itemsize
        delta = TYPES[case["delta"]].itemsize
        gate = {"none": 0, "channels": 4 * H, "rows": T * H * delta}[case["gate"]]
        return {"bytes": T * H * (2 * TYPES[case["stream"]].itemsize + delta) + gate + 4 * H * (2 if case["post"] else 1) + out,
                "flops": T * H * (11 if case["post"] else 7)}
    K = case["K"]
    return {"bytes": T * K * (TYPES[case["dtype"]].itemsize + 1) + 4 * (T if case["block"] == 1 else _groups(T)) * _groups(K),
            "flops": 3 * T * K}


# ------------------------------------------------------------------ in 64 bits, from the definitions
def _values(q, s, block):
    """What a quantised matrix stands for."""
    rows = torch.arange(q.shape[0], device=q.device) // block
    columns = torch.arange(q.shape[1], device=q.device) // 128
    return q.to(torch.float64) * s.to(torch.float64)[rows][:, columns]


def _codes(v, block):
    """(values over their scale, not rounded, scales) of a matrix in 64 bits."""
    T, K = v.shape
    rows, columns = torch.arange(T, device=v.device) // block, torch.arange(K, device=v.device) // 128
    at = rows[:, None] * _groups(K) + columns[None, :]
    count = (int(rows[-1]) + 1) * _groups(K)
    a = torch.zeros(count, dtype=torch.float64, device=v.device).scatter_reduce_(0, at.reshape(-1), v.abs().reshape(-1), "amax")
    s = torch.maximum(a / 448, torch.full_like(a, TINY))
    return v / s[at], s.view(-1, _groups(K))


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        return _values(st["x"], st["x_scales"], 1) @ _values(st["w"], st["w_scales"], 128).t()
    if op == "gated":
        x = _values(st["x"], st["x_scales"], 1)
        g = x @ _values(st["gate"], st["gate_scales"], 128).t()
        u = x @ _values(st["up"], st["up_scales"], 128).t()
        return _codes(g * torch.sigmoid(g) * u, 1)
    if op == "norms":
        d = st["d"].to(torch.float64)
        if case["post"]:
            d = d * torch.rsqrt((d * d).mean(1, keepdim=True) + 1e-6) * st["post_weight"].to(torch.float64)
        if st["g"] is not None:
            d = d * st["g"].to(torch.float64)
        x = st["x"].to(torch.float64) + st["c"] * d
        kept = x.to(st["x"].dtype).to(torch.float64)
        h = kept * torch.rsqrt((kept * kept).mean(1, keepdim=True) + 1e-6) * st["weight"].to(torch.float64)
        return [x, *_codes(h, 1)] if case["out"] == "fp8" else [x, h]
    return _codes(st["x"].to(torch.float64), case["block"])
