"""What is measured of the operators around the sampler, and their plain forms.

Two operators: ``verify``, the verification of drafted tokens against the target model's probabilities
(speculative decoding; the random numbers are inputs), and ``head``, the product of hidden states with a
4-bit weight matrix with group scales that makes the logits the sampler and the verification read.

``run`` computes a case in its plain form (elementary torch operations) or, where ``own`` is true, through
the package's entry points.  Sizes: the vocabularies are those of the sampler's workloads (32000, 128256,
151936, 262144), the batch of 64 sequences is that of its headline workload; hidden sizes are generic.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
# residual masses up to this are rounding noise of p - q: the draw is then made from p itself
EMPTY_RESIDUAL = 2.0 ** -30


def _verify(name, sequences, drafts, vocab, dtype, temperature, draft_model=True, ragged=False, pad=0):
    return {"name": name, "op": "verify", "sequences": sequences, "drafts": drafts, "vocab": vocab, "dtype": dtype,
            "temperature": temperature, "draft_model": draft_model, "ragged": ragged, "pad": pad}


def _head(name, rows, vocab, hidden, group, dtype, logits, zeros=False, scales=None):
    return {"name": name, "op": "head", "rows": rows, "vocab": vocab, "hidden": hidden, "group": group, "dtype": dtype,
            "logits": logits, "zeros": zeros, "scales": scales or dtype}


def listed():
    return [
        # one user's sequence on a small vocabulary: the latency of a single call
        _verify("verify_1x4_32000_f32", 1, 4, 32000, "f32", 0.8),
        # the headline serving batch, four drafts of a draft model each
        _verify("verify_64x4_128256_bf16", 64, 4, 128256, "bf16", 0.6),
        # a ragged batch: every sequence with a draft length and a temperature of its own, rows padded
        _verify("verify_33x7_151936_f16_ragged", 33, 7, 151936, "f16", 1.0, ragged=True, pad=5),
        # drafts looked up in the prompt (no draft probabilities) on the largest vocabulary
        _verify("verify_16x5_262144_bf16_lookup", 16, 5, 262144, "bf16", 0.7, draft_model=False),
        # greedy serving: drafts are kept while they are the target's arg-max
        _verify("verify_64x4_128256_bf16_greedy", 64, 4, 128256, "bf16", 0.0),
        # one token's logits, small and large model
        _head("head_1_32000x2048_g32_bf16", 1, 32000, 2048, 32, "bf16", "bf16"),
        _head("head_1_128256x4096_g128_bf16", 1, 128256, 4096, 128, "bf16", "bf16"),
        # the target's logits for one sequence's four drafts, asymmetric weights, logits kept in 32 bits
        _head("head_5_151936x5120_g64_f16_zeros", 5, 151936, 5120, 64, "f16", "f32", zeros=True),
        # a decode step in 32 bits with sizes that divide nothing
        _head("head_3_50257x1601_g32_f32", 3, 50257, 1601, 32, "f32", "f32"),
        # the headline serving batch: one token a sequence
        _head("head_64_128256x4096_g128_bf16", 64, 128256, 4096, 128, "bf16", "bf16"),
        # ... and a verification step of it: four drafts and the token before them
        _head("head_320_128256x4096_g128_bf16", 320, 128256, 4096, 128, "bf16", "bf16"),
        # a batch that fills no tile, 32-column groups
        _head("head_37_32000x4096_g32_f16", 37, 32000, 4096, 32, "f16", "f16"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    if rng.random() < 0.5:
        vocab = _log_int(rng, 1000, 262144)
        drafts = rng.randint(1, 8)
        dtype = rng.choice(["f32", "f16", "bf16"])
        most = 64 * 9 * 128256 * 2 // (SIZES[dtype] * (2 * drafts + 1) * vocab)
        return _verify(None, _log_int(rng, 1, max(1, min(256, most))), drafts, vocab, dtype,
                       rng.choice([0.0, 0.3, 0.6, 0.8, 1.0, 1.3]), draft_model=rng.random() < 0.7, ragged=rng.random() < 0.5,
                       pad=rng.choice([0, 0, 1, 8, 13]))
    hidden = _log_int(rng, 64, 8192)
    vocab = _log_int(rng, 1000, min(262144, 128256 * 4096 // hidden))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    return _head(None, _log_int(rng, 1, 320 if dtype != "f32" else 64), vocab, hidden, rng.choice([32, 64, 128, 256]), dtype,
                 rng.choice(["f32", dtype]), zeros=rng.random() < 0.4, scales=rng.choice(["f32", dtype]))


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _verify_inputs(case, seed):
    g = _generator(seed)
    S, K, V = case["sequences"], case["drafts"], case["vocab"]
    dtype, dev = DTYPES[case["dtype"]], "cuda"
    width = V + case["pad"]
    # peaked rows, as a trained model gives them: a normal bulk and a few raised tokens
    target = torch.empty((S, K + 1, width), dtype=torch.float32, device=dev).normal_(generator=g)
    hot = torch.randint(0, V, (S, K + 1, 20), generator=g, device=dev)
    target.scatter_add_(2, hot, torch.full_like(hot, 8, dtype=torch.float32) +
                        2 * torch.empty(hot.shape, dtype=torch.float32, device=dev).normal_(generator=g))
    temperatures = torch.full((S,), case["temperature"], dtype=torch.float32, device=dev)
    lengths = None
    if case["ragged"]:
        lengths = torch.randint(0, K + 1, (S,), generator=g, device=dev).to(torch.int32)
        temperatures *= 0.5 + torch.rand((S,), generator=g, device=dev)
    # the draft model sees about the same: its rows are the target's with noise
    draft = target[:, :K] + 0.5 * torch.empty((S, K, width), dtype=torch.float32, device=dev).normal_(generator=g)
    draft, target = draft.to(dtype)[:, :, :V], target.to(dtype)[:, :, :V]
    # drafts drawn from the draft model at the same temperature (the arg-max of logits with Gumbel noise)
    noise = torch.empty((S, K, V), dtype=torch.float32, device=dev).exponential_(generator=g).log_()
    heat = (temperatures if case["draft_model"] else 0.5 * temperatures)[:, None, None]
    tokens = (draft.float() - heat * noise).argmax(2).to(torch.int32)
    coins = torch.rand((S, K + 1), generator=g, device=dev)
    return {"target": target, "draft": draft if case["draft_model"] else None, "tokens": tokens, "lengths": lengths,
            "temperatures": temperatures, "coins": coins}


def _head_inputs(case, seed):
    g = _generator(seed)
    M, V, D, group = case["rows"], case["vocab"], case["hidden"], case["group"]
    dev = "cuda"
    groups = (D + group - 1) // group
    packed = torch.randint(0, 256, (V, (D + 1) // 2), generator=g, device=dev, dtype=torch.uint8)
    scales = (0.004 * (0.5 + torch.rand((V, groups), generator=g, device=dev))).to(DTYPES[case["scales"]])
    zeros = None
    if case["zeros"]:
        zeros = (0.01 * torch.empty((V, groups), device=dev).normal_(generator=g)).to(DTYPES[case["scales"]])
    # the final norm's output: unit variance, some channels far above it
    hidden = torch.empty((M, D), device=dev).normal_(generator=g)
    hidden[:, torch.randint(0, D, (max(1, D // 512),), generator=g, device=dev)] *= 20
    return {"hidden": hidden.to(DTYPES[case["dtype"]]), "packed": packed, "scales": scales, "zeros": zeros, "group": group,
            "columns": D, "logits": DTYPES[case["logits"]]}


def prepare(case, seed):
    if case["op"] == "verify":
        state = _verify_inputs(case, seed)
        state["op"] = "verify"
        if own:
            import executorch_amd as ea
            state["verifier"] = ea.DraftVerifier(case["vocab"], case["sequences"], case["drafts"])
        return state
    state = _head_inputs(case, seed)
    state["op"] = "head"
    if own:  # a program lays its weights out once and keeps that form
        import executorch_amd as ea
        state["head"] = ea.LogitHead(state["packed"], state["scales"], state["group"], hidden_size=state["columns"],
                                     zeros=state["zeros"])
        state["packed"] = state["scales"] = state["zeros"] = None
    return state


def run(state):
    if state["op"] == "verify":
        if own:
            return state["verifier"].verify(state["target"], state["tokens"], state["coins"], draft_logits=state["draft"],
                                            draft_lengths=state["lengths"], temperature=state["temperatures"])
        return _plain_verify(state["target"], state["draft"], state["tokens"], state["lengths"], state["temperatures"], state["coins"])
    if own:
        return state["head"].logits(state["hidden"], dtype=state["logits"])
    return _plain_head(state["hidden"], state["packed"], state["scales"], state["zeros"], state["group"], state["columns"], state["logits"])


def _plain_head(hidden, packed, scales, zeros, group, columns, dtype):
    # weight[v, k] = (nibble - 8) * scale[v, k // group] + zero[v, k // group]; even columns in the low nibbles
    nibbles = torch.stack((packed & 15, packed >> 4), dim=2).reshape(packed.shape[0], -1)[:, :columns]
    which = torch.arange(columns, device=packed.device) // group
    weight = (nibbles.float() - 8) * scales.float()[:, which]
    if zeros is not None:
        weight += zeros.float()[:, which]
    return (hidden.float() @ weight.t()).to(dtype)


def _plain_verify(target, draft, tokens, lengths, temperatures, coins):
    S, positions, V = target.shape
    K = positions - 1
    dev = target.device
    ids = torch.arange(V, device=dev)
    greedy = temperatures == 0
    heat = torch.where(greedy, 1, temperatures).double()[:, None, None]

    def probabilities(logits):
        x = logits.double()
        w = torch.exp((x - x.amax(2, keepdim=True)) / heat)
        return w / w.sum(2, keepdim=True)

    # 64 bits throughout: a coin may fall next to a border between two tokens
    p = probabilities(target)
    top = target.amax(2, keepdim=True)
    best = torch.where(target == top, ids, V).amin(2)  # the first of equal maxima
    inside = torch.arange(K, device=dev) < (K if lengths is None else lengths[:, None])
    at = tokens.long()[:, :, None]
    p_token = p[:, :K].gather(2, at)[:, :, 0]
    if draft is not None:
        q = probabilities(draft)
        q_token = q.gather(2, at)[:, :, 0]
    else:
        q, q_token = None, torch.ones_like(p_token)
    keep = torch.where(greedy[:, None], tokens == best[:, :K], coins[:, :K].double() * q_token < p_token) & inside
    kept = keep.long().cumprod(1).sum(1)
    every = torch.arange(S, device=dev)
    rejected = kept < (K if lengths is None else lengths)
    slot = kept.clamp(max=K - 1)
    row = p[every, kept]
    if draft is not None:
        taken = q[every, slot]
    else:
        taken = (ids == tokens[every, slot, None]).double()
    rest = (row - taken).clamp(min=0)
    use_rest = rejected & (rest.sum(1) > EMPTY_RESIDUAL)
    weights = torch.where(use_rest[:, None], rest, row)
    sums = weights.cumsum(1)
    drawn = (sums <= coins[:, K:].double() * sums[:, -1:]).sum(1)
    last = torch.where(weights > 0, ids, 0).amax(1)
    drawn = torch.where(greedy, best[every, kept], torch.minimum(drawn, last))
    column = torch.arange(positions, device=dev)
    padded = torch.cat((tokens.long(), tokens.new_zeros((S, 1)).long()), 1)
    out = torch.where(column < kept[:, None], padded, torch.where(column == kept[:, None], drawn[:, None], -1))
    return out.to(torch.int32), kept.to(torch.int32)


def work(case):
    if case["op"] == "verify":
        S, K, V = case["sequences"], case["drafts"], case["vocab"]
        mean = K / 2 if case["ragged"] else K
        entries = S * (mean + 1) * V
        if case["draft_model"] and case["temperature"] != 0:
            entries += S * mean * V
        return {"bytes": entries * SIZES[case["dtype"]] + S * (12 * K + 16), "flops": entries * (6 if case["temperature"] else 1)}
    M, V, D = case["rows"], case["vocab"], case["hidden"]
    groups = (D + case["group"] - 1) // case["group"]
    return {"bytes": V * ((D + 1) // 2) + V * groups * SIZES[case["scales"]] * (2 if case["zeros"] else 1) +
            M * D * SIZES[case["dtype"]] + M * V * SIZES[case["logits"]], "flops": 2 * M * V * D}


def exact(case, seed):
    if case["op"] == "verify":
        return _exact_verify(_verify_inputs(case, seed))
    s = _head_inputs(case, seed)
    V, D, group = case["vocab"], case["hidden"], case["group"]
    x = s["hidden"].double()
    out = torch.empty((case["rows"], V), dtype=torch.float64, device=x.device)
    # sum over groups of scale * (sum of x * nibble - 8 * sum of x) + zero * sum of x, some vocabulary rows at a time
    step = max(1, (1 << 28) // D)
    for v in range(0, V, step):
        byte = s["packed"][v:v + step].to(torch.int16)
        n = byte.new_empty((byte.shape[0], byte.shape[1] * 2))
        n[:, 0::2], n[:, 1::2] = byte % 16, byte // 16
        part = torch.zeros((x.shape[0], byte.shape[0]), dtype=torch.float64, device=x.device)
        for k in range(0, D, group):
            xs = x[:, k:k + group]
            ns = n[:, k:min(D, k + group)].double()
            sums = xs.sum(1, keepdim=True)
            part += s["scales"][v:v + step, k // group].double() * (xs @ ns.t().contiguous() - 8 * sums)
            if s["zeros"] is not None:
                part += s["zeros"][v:v + step, k // group].double() * sums
        out[:, v:v + step] = part
    return out


def _exact_verify(s):
    """Sequence by sequence and position by position, in logarithms."""
    S, K = s["tokens"].shape
    tokens, kept = [], []
    drafted = s["tokens"].tolist()
    coins = s["coins"].double().tolist()
    heats = s["temperatures"].double().tolist()
    lengths = [K] * S if s["lengths"] is None else s["lengths"].tolist()
    for b in range(S):
        line, n, final = [], 0, None
        while final is None:
            row = s["target"][b, n].double()
            reject = n < lengths[b]
            if heats[b] == 0:
                final = int((row == row.max()).nonzero()[0, 0])
                if reject and drafted[b][n] == final:
                    final = None
            else:
                logp = torch.log_softmax(row / heats[b], 0)
                logq = None
                x = drafted[b][n] if reject else -1
                if reject and s["draft"] is not None:
                    logq = torch.log_softmax(s["draft"][b, n].double() / heats[b], 0)
                if reject:
                    limit = float(logp[x]) - (float(logq[x]) if logq is not None else 0.0)
                    accept = coins[b][n] == 0 and limit > -math.inf or coins[b][n] > 0 and math.log(coins[b][n]) < limit
                else:
                    accept = False
                if not accept:
                    mass = logp.exp()
                    if reject:
                        rest = mass.clone()
                        if logq is not None:
                            rest -= logq.exp()
                        else:
                            rest[x] = 0
                        rest[rest < 0] = 0
                        if float(rest.sum()) > EMPTY_RESIDUAL:
                            mass = rest
                    ladder = torch.cumsum(mass, 0)
                    level = ladder[-1:] * coins[b][K]
                    final = int(torch.searchsorted(ladder, level, right=True)[0])
                    final = min(final, int(mass.nonzero()[-1, 0]))
            if final is None:
                line.append(drafted[b][n])
                n += 1
        tokens.append(line + [final] + [-1] * (K - n))
        kept.append(n)
    dev = s["target"].device
    return torch.tensor(tokens, dtype=torch.int32, device=dev), torch.tensor(kept, dtype=torch.int32, device=dev)
