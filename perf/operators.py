"""The operators of serving from a paged cache, in their plain form and as this library's calls: rotary positions, the append
of new keys and values to pages, and the attention of new tokens (one a sequence or a chunk) over the pages.

A cache is [pages][kv heads][page size][head dim]; sequence b holds lens[b] positions, position p of it lies in page
pages[b][p // page size], slot p % page size.  The new tokens of all sequences stand behind one another, those of sequence b
are rows starts[b] .. starts[b + 1], and they are the last positions of their sequence.

listed() names the cases, draw() gives more of the same ranges, prepare() makes what a program holds before the call,
run() is the call, work() the bytes and operations that it cannot do without, exact() the same result in 64 bits."""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _attention(name, dtype, heads, kv_heads, page, seqs, chunks, chunk, hist, head_dim=128, window=0, alibi=False, left=False):
    """`chunks` of the `seqs` sequences bring chunk[0] .. chunk[1] tokens, the others one; each has hist[0] .. hist[1]
    tokens in the cache before.  left: the first positions of some sequences are padding."""
    return {"name": name, "op": "paged_mha", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "seqs": seqs, "chunks": chunks, "chunk_min": chunk[0], "chunk_max": chunk[1], "hist_min": hist[0],
            "hist_max": hist[1], "window": window, "alibi": alibi, "left": left}


def _store(name, dtype, heads, kv_heads, page, seqs, chunks, chunk, hist, rotary_dim, interleaved, scaling):
    return {"name": name, "op": "paged_store", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": 128,
            "page": page, "seqs": seqs, "chunks": chunks, "chunk_min": chunk[0], "chunk_max": chunk[1], "hist_min": hist[0],
            "hist_max": hist[1], "rotary_dim": rotary_dim, "interleaved": interleaved, "scaling": scaling}


def _rotary(name, dtype, tokens, heads, kv_heads, rotary_dim, interleaved, scaling, far, head_dim=128):
    return {"name": name, "op": "rotary", "dtype": dtype, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "rotary_dim": rotary_dim, "interleaved": interleaved, "scaling": scaling, "far": far}


def listed():
    return [
        # one user's next token after a short exchange: latency alone
        _attention("mha_one_short", "fp16", 32, 32, 16, 1, 0, (1, 1), (300, 300)),
        # a decode step of a batch whose sequences have very different ages, shared heads
        _attention("mha_batch_of_64", "bf16", 32, 8, 64, 64, 0, (1, 1), (200, 8000)),
        # two users with whole books in the cache, the 65B width's heads in groups of eight
        _attention("mha_two_books", "fp16", 64, 8, 16, 2, 0, (1, 1), (60000, 100000)),
        # a handful of guessed tokens checked at once for each of 16 sequences
        _attention("mha_check_guesses", "fp16", 32, 8, 16, 16, 16, (5, 5), (1000, 3000)),
        # one chunk of a long prompt, the earlier chunks in the cache already
        _attention("mha_chunk", "bf16", 32, 8, 16, 1, 1, (512, 512), (8192, 8192)),
        # what a scheduler hands over in one step: a chunk of one prompt beside the next tokens of other users; ALiBi, 13B width
        _attention("mha_mixed", "fp16", 40, 40, 32, 24, 1, (777, 777), (100, 4000), alibi=True),
        # a long chunk late in a very long prompt: the most arithmetic
        _attention("mha_long_chunk", "bf16", 64, 8, 64, 1, 1, (1024, 1024), (24000, 24000)),
        # short heads, a sliding window, some padding on the left, odd lengths
        _attention("mha_window", "fp16", 16, 2, 16, 3, 3, (100, 601), (0, 5000), head_dim=64, window=1000, left=True),
        # a decode step of eight users: rotating the new queries and keys
        _rotary("rotary_step", "fp16", 8, 32, 32, 128, False, "none", 2000),
        # a batch of chunks, half of each head rotated, far positions, frequencies stretched for long contexts
        _rotary("rotary_far", "bf16", 6001, 40, 8, 64, True, "yarn", 120000),
        # the append of one token for each of 64 sequences, with the rotation
        _store("store_step", "fp16", 32, 8, 16, 64, 0, (1, 1), (20, 400), 128, False, "bands"),
        # the append of ragged chunks of five prompts at the 13B width
        _store("store_chunks", "fp16", 40, 40, 32, 5, 5, (300, 2000), (0, 1000), 128, False, "linear"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("paged_mha", "paged_mha", "paged_mha", "paged_mha", "rotary", "paged_store"))
    dtype = rng.choice(("fp16", "bf16"))
    page = rng.choice((16, 32, 64, 128))
    scaling = rng.choice(("none", "linear", "bands", "yarn"))
    if op == "rotary":
        heads, kv_heads = rng.choice(((32, 32), (32, 8), (40, 40), (40, 8), (64, 8)))
        c = _rotary("", dtype, _log_int(rng, 1, 6000), heads, kv_heads, rng.choice((32, 64, 96, 128)), rng.random() < 0.5,
                    scaling, _log_int(rng, 100, 1000000))
    elif op == "paged_store":
        heads, kv_heads = rng.choice(((32, 32), (32, 8), (40, 8), (64, 8)))
        seqs = _log_int(rng, 1, 64)
        chunks = rng.choice((0, 1, seqs))
        top = _log_int(rng, 2, max(2, 6000 // max(1, chunks)))
        c = _store("", dtype, heads, kv_heads, page, seqs, chunks, (1 + top // 2, top), (0, _log_int(rng, 10, 400)),
                   rng.choice((32, 64, 128)), rng.random() < 0.5, scaling)
    else:
        heads, kv_heads = rng.choice(((32, 32), (32, 8), (40, 40), (40, 8), (64, 8), (28, 4), (32, 1), (16, 16)))
        kind = rng.choice(("step", "step", "guesses", "chunk", "mixed"))
        seqs = {"step": _log_int(rng, 1, 64), "guesses": _log_int(rng, 1, 32), "chunk": rng.choice((1, 1, 2, 3)),
                "mixed": _log_int(rng, 2, 32)}[kind]
        chunks = {"step": 0, "guesses": seqs, "chunk": seqs, "mixed": 1}[kind]
        top = {"step": 1, "guesses": rng.randint(2, 16), "chunk": _log_int(rng, 20, 1000), "mixed": _log_int(rng, 20, 700)}[kind]
        # what the plain form holds at once is all scores: heads x tokens x keys of all sequences
        room = 1.2e9 / heads / (chunks * top + seqs - chunks)
        keys = int(min(60000, max(200, room / seqs - top)))
        far = _log_int(rng, 100, keys)
        c = _attention("", dtype, heads, kv_heads, page, seqs, chunks, (1 + top // 2, top), (rng.choice((0, far // 20)), far),
                       head_dim=rng.choice((64, 128, 128)), window=rng.choice((0, 0, 0, _log_int(rng, 10, 4000))),
                       alibi=rng.random() < 0.2, left=rng.random() < 0.2)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------------------
# the shape of a case: it follows from the case alone
# ---------------------------------------------------------------------------------------------------------------------
def _lengths(c):
    """(new tokens, positions in the cache with them, first position that counts) of each sequence."""
    rng = random.Random("%d %d %d %d %d" % (c["seqs"], c["chunks"], c["chunk_max"], c["hist_min"], c["hist_max"]))
    place = list(range(c["seqs"]))
    rng.shuffle(place)
    new = [rng.randint(c["chunk_min"], c["chunk_max"]) if n < c["chunks"] else 1 for n in place]
    lens = [_log_int(rng, c["hist_min"] + 1, c["hist_max"] + 1) - 1 + n for n in new]
    first = [rng.randint(0, x) // 3 if c.get("left") and n % 2 == 0 else 0 for n, x in zip(place, lens)]
    return new, lens, first


def _visible(c):
    """Key positions read at least once, and pairs of a new token and a key that it sees."""
    low = lambda p, first: max(first, p - c["window"] + 1 if c["window"] else 0)  # noqa: E731
    seqs = list(zip(*_lengths(c)))
    read = sum(max(0, x - low(x - n, first)) for n, x, first in seqs)
    return read, sum(max(0, p + 1 - low(p, first)) for n, x, first in seqs for p in range(x - n, x))


def work(case):
    H, K, D = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rotary":
        rows = case["tokens"] * (H + K)
        return {"bytes": 2 * 2 * rows * D + 8 * case["tokens"], "flops": 3 * rows * case["rotary_dim"]}
    tokens = sum(_lengths(case)[0])
    if case["op"] == "paged_store":
        return {"bytes": 2 * 2 * tokens * (H + 2 * K) * D, "flops": 3 * tokens * (H + K) * case["rotary_dim"]}
    read, pairs = _visible(case)
    return {"bytes": 2 * 2 * read * K * D + 2 * 2 * tokens * H * D, "flops": 4 * pairs * H * D}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _frequencies(dim, scaling):
    """Radians a position for each pair of a head's rotated part, and the factor on the rotated values."""
    base, factor, original = 10000.0, 8.0, 4096.0
    freqs, magnitude = [base ** (-2.0 * i / dim) for i in range(dim // 2)], 1.0
    if scaling == "linear":
        freqs = [f / factor for f in freqs]
    elif scaling == "bands":     # short waves as they are, long ones stretched, a blend between
        low, high = 1.0, 4.0
        def bands(f):
            turns = original * f / (2 * math.pi)
            s = min(1.0, max(0.0, (turns - low) / (high - low)))
            return s * f + (1 - s) * f / factor
        freqs = [bands(f) for f in freqs]
    elif scaling == "yarn":
        place = lambda turns: dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(0, math.floor(place(32.0))), min(dim - 1, math.ceil(place(1.0)))
        s = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(dim // 2)]
        freqs = [f / factor * x + f * (1 - x) for f, x in zip(freqs, s)]
        magnitude = 0.1 * math.log(factor) + 1.0
    return freqs, magnitude


def _slopes(heads):
    n = 2 ** math.floor(math.log2(heads))
    s = [2.0 ** (-8.0 * (i + 1) / n) for i in range(n)]
    return s + [2.0 ** (-4.0 * (2 * i + 1) / n) for i in range(heads - n)]


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype, H, K, D = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["head_dim"]
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)  # noqa: E731
    s = {"case": case}
    if case["op"] != "paged_mha":
        freqs, s["magnitude"] = _frequencies(case["rotary_dim"], case["scaling"])
        s["freqs"] = torch.tensor(freqs, dtype=torch.float64, device="cuda")
    if case["op"] == "rotary":
        n = case["tokens"]
        qkv = randn(n, (H + 2 * K) * D)          # the fused projection of a model: q and k are views of it
        s["q"], s["k"] = qkv[:, :H * D].view(n, H, D), qkv[:, H * D:(H + K) * D].view(n, K, D)
        s["positions"] = torch.randint(0, case["far"], (n,), generator=gen, device="cuda")
        return s
    new, lens, first = _lengths(case)
    P, n = case["page"], sum(new)
    need = [-(-x // P) for x in lens]
    total = sum(need) + 7
    s["k_cache"], s["v_cache"] = randn(total, K, P, D), randn(total, K, P, D)
    width = max(need) + 1
    owner = torch.tensor([b for b, k in enumerate(need) for _ in range(k)], device="cuda")
    column = torch.tensor([j for k in need for j in range(k)], device="cuda")
    s["pages"] = torch.zeros(len(new), width, dtype=torch.int32, device="cuda")
    s["pages"][owner, column] = torch.randperm(total, generator=gen, device="cuda")[:sum(need)].int()
    s["starts"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["total_len"], s["max_tokens"], s["max_len"] = sum(lens), max(new), max(lens)
    if case["op"] == "paged_store":
        qkv = randn(n, (H + 2 * K) * D)
        s["q"], s["k"] = qkv[:, :H * D].view(n, H, D), qkv[:, H * D:(H + K) * D].view(n, K, D)
        s["v"] = qkv[:, (H + K) * D:].view(n, K, D)
        return s
    s["q"] = 2 * randn(n, H, D)                  # scores of a few units: some keys count, most hardly do
    s["first_key"] = torch.tensor(first, dtype=torch.int32, device="cuda") if case["left"] else None
    s["alibi_slopes"] = torch.tensor(_slopes(H), dtype=torch.float32, device="cuda") if case["alibi"] else None
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _tokens(s, n):
    """Sequence and position of each new token."""
    row = torch.arange(n, device="cuda")
    seq = torch.searchsorted(s["starts"][1:].contiguous(), row.int(), right=True)
    return seq, s["lens"][seq].long() - s["starts"][seq + 1] + row


def _rotated(x, positions, freqs, interleaved, magnitude):
    angle = positions.double()[:, None] * freqs
    cos, sin = ((f(angle) * magnitude).float()[:, None, :] for f in (torch.cos, torch.sin))
    r = 2 * freqs.numel()
    y = x.float()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., :r // 2], y[..., r // 2:r])
    pair = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
    return torch.cat((turned, y[..., r:]), -1).to(x.dtype)


def _plain_rotary(s):
    turn = lambda x: _rotated(x, s["positions"], s["freqs"], s["case"]["interleaved"], s["magnitude"])  # noqa: E731
    return turn(s["q"]), turn(s["k"])


def _plain_store(s):
    seq, pos = _tokens(s, s["q"].shape[0])
    turn = lambda x: _rotated(x, pos, s["freqs"], s["case"]["interleaved"], s["magnitude"])  # noqa: E731
    P = s["k_cache"].shape[2]
    page, slot = s["pages"][seq, pos // P].long(), pos % P
    s["k_cache"][page, :, slot] = turn(s["k"])
    s["v_cache"][page, :, slot] = s["v"]
    return turn(s["q"]), s["k_cache"], s["v_cache"]


def _plain_mha(s):
    c, q = s["case"], s["q"]
    n, H, D = q.shape
    K, P = s["k_cache"].shape[1:3]
    seq, pos = _tokens(s, n)
    # the keys of all sequences behind one another
    ends = torch.cumsum(s["lens"], 0)
    key = torch.arange(s["total_len"], device="cuda")
    kseq = torch.searchsorted(ends, key, right=True)
    kpos = key - ends[kseq] + s["lens"][kseq]
    page, slot = s["pages"][kseq, kpos // P].long(), kpos % P
    k, v = (s[w][page, :, slot].float().transpose(0, 1) for w in ("k_cache", "v_cache"))      # [kv heads][keys][D]
    scores = torch.matmul(q.float().view(n, K, H // K, D).permute(1, 2, 0, 3).reshape(K, H // K * n, D), k.transpose(1, 2))
    scores = scores.mul_(1 / math.sqrt(D)).view(K, H // K, n, -1)
    if s["alibi_slopes"] is not None:
        scores += s["alibi_slopes"].view(K, H // K, 1, 1) * (kpos[None, :] - pos[:, None]).float()
    seen = (kseq[None, :] == seq[:, None]) & (kpos[None, :] <= pos[:, None])
    if c["window"]:
        seen &= kpos[None, :] > pos[:, None] - c["window"]
    if s["first_key"] is not None:
        seen &= kpos[None, :] >= s["first_key"][seq][:, None]
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_(min=-1e30)      # a row that sees nothing: no probabilities, zeros
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(K, H // K * n, -1), v).view(K, H // K, n, D) / total.clamp_(min=1e-30)
    return out.permute(2, 0, 1, 3).reshape(n, H, D).to(q.dtype)


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"rotary": _plain_rotary, "paged_store": _plain_store, "paged_mha": _plain_mha}[c["op"]](s)
    from eet_b200 import paged
    if c["op"] == "rotary":
        return paged.apply_rotary(s["q"], s["k"], s["positions"], s["freqs"], interleaved=c["interleaved"],
                                  magnitude=s["magnitude"])
    if c["op"] == "paged_store":
        q = paged.paged_store(s["k"], s["v"], s["k_cache"], s["v_cache"], s["pages"], s["starts"], s["lens"], q=s["q"],
                              freqs=s["freqs"], interleaved=c["interleaved"], magnitude=s["magnitude"])
        return q, s["k_cache"], s["v_cache"]
    return paged.paged_mha(s["q"], s["k_cache"], s["v_cache"], s["pages"], s["starts"], s["lens"], max_tokens=s["max_tokens"],
                           max_len=s["max_len"], window=c["window"], first_key=s["first_key"],
                           alibi_slopes=s["alibi_slopes"])


# ---------------------------------------------------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------------------------------------------------
def _turn64(x, position, s):
    """Pair i of a row as a complex number, turned by magnitude * exp(i position freqs[i])."""
    x, half = x.double(), s["freqs"].numel()
    phase = torch.polar(torch.full((len(x), half), float(s["magnitude"]), dtype=torch.float64, device="cuda"),
                        torch.outer(position.double(), s["freqs"]))[:, None]
    y = x.clone()
    places = torch.arange(2 * half, device="cuda")
    one, two = (places[0::2], places[1::2]) if s["case"]["interleaved"] else (places[:half], places[half:])
    z = torch.complex(x[..., one], x[..., two]) * phase
    y[..., one], y[..., two] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return tuple(_turn64(s[w], s["positions"], s) for w in ("q", "k"))
    new, lens, first = _lengths(case)
    P, at = case["page"], 0
    if case["op"] == "paged_store":
        q = s["q"].double()
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        for b, n in enumerate(new):
            place = torch.arange(lens[b] - n, lens[b], device="cuda")
            page = s["pages"][b].long()[place // P]
            q[at:at + n] = _turn64(s["q"][at:at + n], place, s)
            kc[page, :, place % P] = _turn64(s["k"][at:at + n], place, s)
            vc[page, :, place % P] = s["v"][at:at + n].double()
            at += n
        return q, kc, vc
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    G, D = case["heads"] // case["kv_heads"], case["head_dim"]
    for b, n in enumerate(new):
        place = torch.arange(lens[b], device="cuda")
        page = s["pages"][b].long()[place // P]
        for h in range(case["kv_heads"]):
            k, v = (s[w][page, h, place % P].double() for w in ("k_cache", "v_cache"))
            for i in range(0, n, 256):
                rows = slice(at + i, at + min(i + 256, n))
                p = torch.arange(lens[b] - n + i, lens[b] - n + min(i + 256, n), device="cuda")
                seen = (place <= p[:, None]) & (place >= first[b])
                if case["window"]:
                    seen &= place + case["window"] > p[:, None]
                for g in range(G):
                    head = h * G + g
                    x = s["q"][rows, head].double() @ k.T / D ** 0.5
                    if case["alibi"]:
                        x += s["alibi_slopes"][head].double() * (place - p[:, None])
                    weights = torch.softmax(x.masked_fill(~seen, -1e300), -1) * seen
                    out[rows, head] = weights @ v
        at += n
    return out
