"""The operators of serving from an 8-bit paged cache up to the next token, in their plain form and as this library's calls: the
append of new keys and values as codes and scales, reading them back, the attention of new tokens (one a sequence or a chunk) over
such pages, and the choice of the next token with temperature, top-k, top-p and min-p from given random numbers.

A cache is codes [pages][kv heads][page size][head dim], int8 or e4m3, with a scale [pages][kv heads][page size] for each row of
head dim; a value is its code times the scale of its row.  Sequence b holds lens[b] positions, position p of it lies in page
pages[b][p // page size], slot p % page size.  The new tokens of all sequences stand behind one another, those of sequence b are
rows starts[b] .. starts[b + 1], and they are the last positions of their sequence.

listed() names the cases, draw() gives more of the same ranges, prepare() makes what a program holds before the call, run() is
the call, work() the bytes and operations that it cannot do without, exact() the same result in 64 bits."""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def _attention(name, codes, dtype, heads, kv_heads, page, seqs, chunks, chunk, hist, head_dim=128, window=0, alibi=False, left=False):
    """`chunks` of the `seqs` sequences bring chunk[0] .. chunk[1] tokens, the others one; each has hist[0] .. hist[1]
    tokens in the cache before.  left: the first positions of some sequences are padding."""
    return {"name": name, "op": "mha", "codes": codes, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "seqs": seqs, "chunks": chunks, "chunk_min": chunk[0], "chunk_max": chunk[1], "hist_min": hist[0],
            "hist_max": hist[1], "window": window, "alibi": alibi, "left": left}


def _append(name, codes, dtype, heads, kv_heads, page, seqs, chunks, chunk, hist, rotary_dim, interleaved, head_dim=128):
    return {"name": name, "op": "append", "codes": codes, "dtype": dtype, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "seqs": seqs, "chunks": chunks, "chunk_min": chunk[0], "chunk_max": chunk[1],
            "hist_min": hist[0], "hist_max": hist[1], "rotary_dim": rotary_dim, "interleaved": interleaved}


def _load(name, codes, dtype, kv_heads, page, seqs, hist, head_dim=128):
    """Whole histories of hist[0] .. hist[1] positions are read back."""
    return {"name": name, "op": "load", "codes": codes, "dtype": dtype, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "seqs": seqs, "chunks": seqs, "chunk_min": hist[0], "chunk_max": hist[1], "hist_min": 0, "hist_max": 0}


def _sample(name, dtype, rows, vocab, temperature, top_k, top_p, min_p, mixed=False, banned=False):
    """mixed: every row has settings of its own around these, as the requests of a batch do, some of them greedy.  banned: some
    tokens are masked out with -inf."""
    return {"name": name, "op": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "temperature": temperature, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "mixed": mixed, "banned": banned}


def listed():
    return [
        # one user's next token after a short exchange: latency alone
        _attention("mha_one_short", "int8", "fp16", 32, 32, 16, 1, 0, (1, 1), (300, 300)),
        # a decode step of a batch whose sequences have very different ages, shared heads
        _attention("mha_batch_of_64", "int8", "bf16", 32, 8, 64, 64, 0, (1, 1), (200, 8000)),
        # two users with whole books in the cache, the 65B width's heads in groups of eight
        _attention("mha_two_books", "e4m3", "fp16", 64, 8, 16, 2, 0, (1, 1), (60000, 100000)),
        # one chunk of a long prompt, the earlier chunks in the cache already: the most arithmetic
        _attention("mha_chunk", "int8", "bf16", 32, 8, 16, 1, 1, (512, 512), (8192, 8192)),
        # what a scheduler hands over in one step: a chunk of one prompt beside the next tokens of other users; ALiBi, 13B width
        _attention("mha_mixed", "e4m3", "fp16", 40, 40, 32, 24, 1, (333, 333), (100, 4000), alibi=True),
        # the append of one token for each of 64 sequences, with the rotation, and what the cache then holds of them
        _append("append_step", "int8", "fp16", 32, 8, 16, 64, 0, (1, 1), (20, 400), 128, False),
        # the same for ragged chunks of five prompts at the 13B width
        _append("append_chunks", "e4m3", "bf16", 40, 40, 32, 5, 5, (300, 2000), (0, 1000), 64, True),
        # a shared prefix that another worker asks for
        _load("load_prefix", "int8", "fp16", 8, 16, 1, (777, 777)),
        # histories that leave the cache for the host
        _load("load_histories", "e4m3", "bf16", 8, 64, 12, (500, 9000)),
        # one user's next token, with the usual settings
        _sample("sample_one", "fp32", 1, 32000, 0.8, 50, 0.95, 0.0),
        # the next tokens of a batch of requests, each with settings of its own
        _sample("sample_requests", "fp16", 64, 64000, 1.0, 40, 0.9, 0.05, mixed=True, banned=True),
        # many answers to the same questions, drawn for training: the nucleus alone
        _sample("sample_rollouts", "bf16", 256, 64000, 1.0, 0, 0.95, 0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("mha", "mha", "mha", "append", "load", "sample", "sample"))
    codes, dtype = rng.choice(("int8", "e4m3")), rng.choice(("fp16", "bf16"))
    page = rng.choice((16, 32, 64, 128, 256))
    if op == "sample":
        vocab = _log_int(rng, 500, 130000)
        c = _sample("", rng.choice(("fp16", "bf16", "fp32")), _log_int(rng, 1, min(256, 16000000 // vocab)), vocab,
                    rng.choice((1.0, round(rng.uniform(0.3, 2.0), 2))), rng.choice((0, 0, _log_int(rng, 1, 3000))),
                    rng.choice((1.0, round(rng.uniform(0.1, 0.99), 3))), rng.choice((0.0, 0.0, round(rng.uniform(0.005, 0.3), 3))),
                    mixed=rng.random() < 0.3, banned=rng.random() < 0.3)
    elif op == "load":
        seqs = _log_int(rng, 1, 32)
        top = _log_int(rng, 1, 60000 // seqs)
        c = _load("", codes, dtype, rng.choice((1, 4, 8)), page, seqs, (1 + top // 3, top), head_dim=rng.choice((64, 128, 128)))
    elif op == "append":
        heads, kv_heads = rng.choice(((32, 32), (32, 8), (40, 8), (64, 8)))
        seqs = _log_int(rng, 1, 64)
        chunks = rng.choice((0, 1, seqs))
        top = _log_int(rng, 2, max(2, 6000 // max(1, chunks)))
        c = _append("", codes, dtype, heads, kv_heads, page, seqs, chunks, (1 + top // 2, top), (0, _log_int(rng, 10, 400)),
                    rng.choice((32, 64)), rng.random() < 0.5, head_dim=rng.choice((64, 128, 128)))
    else:
        heads, kv_heads = rng.choice(((32, 32), (32, 8), (40, 40), (40, 8), (64, 8), (28, 4), (32, 1), (16, 16)))
        kind = rng.choice(("step", "step", "guesses", "chunk", "mixed"))
        seqs = {"step": _log_int(rng, 1, 64), "guesses": _log_int(rng, 1, 32), "chunk": rng.choice((1, 1, 2, 3)),
                "mixed": _log_int(rng, 2, 32)}[kind]
        chunks = {"step": 0, "guesses": seqs, "chunk": seqs, "mixed": 1}[kind]
        top = {"step": 1, "guesses": rng.randint(2, 16), "chunk": _log_int(rng, 20, 600), "mixed": _log_int(rng, 20, 400)}[kind]
        # what the plain form holds at once is all scores: heads x tokens x keys of all sequences
        room = 1.2e9 / heads / (chunks * top + seqs - chunks)
        keys = int(min(60000, max(200, room / seqs - top)))
        far = _log_int(rng, 100, keys)
        c = _attention("", codes, dtype, heads, kv_heads, page, seqs, chunks, (1 + top // 2, top), (rng.choice((0, far // 20)), far),
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
    if case["op"] == "sample":
        values = case["rows"] * case["vocab"]
        return {"bytes": values * DTYPES[case["dtype"]].itemsize + 16 * case["rows"], "flops": 4 * values}
    K, D, tokens = case["kv_heads"], case["head_dim"], sum(_lengths(case)[0])
    kept = 2 * K * (D + 4)                       # of a position, in bytes: codes and scales of k and v
    if case["op"] == "load":
        return {"bytes": tokens * (kept + 2 * 2 * K * D), "flops": tokens * 2 * K * D}
    H = case["heads"]
    if case["op"] == "append":
        return {"bytes": tokens * (2 * 2 * H * D + 2 * 2 * K * D + kept + 2 * 2 * K * D),
                "flops": tokens * (3 * (H + K) * case["rotary_dim"] + 3 * 2 * K * D)}
    read, pairs = _visible(case)
    return {"bytes": read * kept + 2 * 2 * tokens * H * D, "flops": 4 * pairs * H * D}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _slopes(heads):
    n = 2 ** math.floor(math.log2(heads))
    s = [2.0 ** (-8.0 * (i + 1) / n) for i in range(n)]
    return s + [2.0 ** (-4.0 * (2 * i + 1) / n) for i in range(heads - n)]


def _cache(codes, shape, gen):
    """Codes as rows of normal values leave them, with scales that differ from row to row."""
    dtype, most = CODES[codes]
    c = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(most / 3.0).clamp_(-most, most)
    c = (c.round_() if codes == "int8" else c).to(dtype)
    scale = torch.rand(shape[:3], generator=gen, device="cuda", dtype=torch.float32).add_(0.5).mul_(3.0 / most)
    return c, scale


def _prepare_sample(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    # what a language model says: most tokens far below a handful of likely ones, some rows surer than others
    x = 2.0 * torch.randn(rows, vocab, generator=gen, device="cuda")
    sure = 0.7 + torch.rand(rows, 1, generator=gen, device="cuda")
    place = (torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda") + 7 * torch.arange(60, device="cuda")) % vocab
    likely = 6.0 + 2.5 * torch.empty(rows, 60, device="cuda").exponential_(generator=gen)
    x = x.scatter(1, place, likely) * sure
    if case["banned"]:
        x[:, torch.randperm(vocab, generator=gen, device="cuda")[:vocab // 3]] = -math.inf
    s = {"case": case, "logits": x.to(DTYPES[case["dtype"]]), "uniform": torch.rand(rows, generator=gen, device="cuda")}
    s.update({w: case[w] for w in ("temperature", "top_k", "top_p", "min_p")})
    if case["mixed"]:
        u = torch.rand(4, rows, generator=gen, device="cuda")
        s["temperature"] = torch.where(u[0] < 0.1, torch.zeros_like(u[0]), case["temperature"] * (0.5 + u[0]))
        s["top_k"] = torch.where(u[1] < 0.3, torch.zeros_like(u[1]), 1 + 2 * case["top_k"] * u[1]).int()
        s["top_p"] = torch.where(u[2] < 0.3, torch.ones_like(u[2]), 0.5 * (case["top_p"] + u[2]))
        s["min_p"] = torch.where(u[3] < 0.6, torch.zeros_like(u[3]), case["min_p"] * u[3])
    return s


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    if case["op"] == "sample":
        return _prepare_sample(case, gen)
    dtype, K, D = DTYPES[case["dtype"]], case["kv_heads"], case["head_dim"]
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)  # noqa: E731
    s = {"case": case}
    new, lens, first = _lengths(case)
    P, n = case["page"], sum(new)
    need = [-(-x // P) for x in lens]
    total = sum(need) + 7
    s["k_cache"], s["k_scale"] = _cache(case["codes"], (total, K, P, D), gen)
    s["v_cache"], s["v_scale"] = _cache(case["codes"], (total, K, P, D), gen)
    width = max(need) + 1
    owner = torch.tensor([b for b, k in enumerate(need) for _ in range(k)], device="cuda")
    column = torch.tensor([j for k in need for j in range(k)], device="cuda")
    s["pages"] = torch.zeros(len(new), width, dtype=torch.int32, device="cuda")
    s["pages"][owner, column] = torch.randperm(total, generator=gen, device="cuda")[:sum(need)].int()
    s["starts"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["tokens"], s["total_len"], s["max_tokens"], s["max_len"] = n, sum(lens), max(new), max(lens)
    if case["op"] == "load":
        return s
    H = case["heads"]
    if case["op"] == "append":
        s["freqs"] = torch.tensor([10000.0 ** (-2.0 * i / case["rotary_dim"]) for i in range(case["rotary_dim"] // 2)],
                                  dtype=torch.float64, device="cuda")
        qkv = randn(n, (H + 2 * K) * D)          # the fused projection of a model: q, k and v are views of it
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


def _rotated(x, positions, freqs, interleaved):
    """In 32 bits, not rounded."""
    angle = positions.double()[:, None] * freqs
    cos, sin = (f(angle).float()[:, None, :] for f in (torch.cos, torch.sin))
    r = 2 * freqs.numel()
    y = x.float()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., :r // 2], y[..., r // 2:r])
    pair = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
    return torch.cat((turned, y[..., r:]), -1)


def _plain_quantize(y, codes):
    dtype, most = CODES[codes]
    top = y.abs().amax(-1)
    # (in 64 bits: 16-bit values over a scale made from one of them often lie on the border of two codes, or next to it)
    scale = torch.where(top > 0, top.double() / most, torch.ones_like(top)).float()
    z = (y.double() / scale[..., None].double()).clamp(-most, most)
    # the distance of two codes: 1, in e4m3 of three bits behind the leading one, down to 2^-6
    step = 1.0 if codes == "int8" else torch.ldexp(torch.ones_like(z), (torch.frexp(z).exponent - 4).clamp(min=-9))
    return (torch.round(z / step) * step).to(dtype), scale


def _plain_values(s, page, slot):
    return tuple((s[w + "_cache"][page, :, slot].float() * s[w + "_scale"][page, :, slot][..., None]) for w in ("k", "v"))


def _plain_append(s):
    c = s["case"]
    seq, pos = _tokens(s, s["tokens"])
    page, slot = s["pages"][seq, pos // c["page"]].long(), pos % c["page"]
    for w, y in (("k", _rotated(s["k"], pos, s["freqs"], c["interleaved"])), ("v", s["v"].float())):
        s[w + "_cache"][page, :, slot], s[w + "_scale"][page, :, slot] = _plain_quantize(y, c["codes"])
    k, v = _plain_values(s, page, slot)
    q = _rotated(s["q"], pos, s["freqs"], c["interleaved"]).to(s["q"].dtype)
    return q, k.to(q.dtype), v.to(q.dtype), s["k_scale"], s["v_scale"]


def _plain_load(s):
    c = s["case"]
    seq, pos = _tokens(s, s["tokens"])
    k, v = _plain_values(s, s["pages"][seq, pos // c["page"]].long(), pos % c["page"])
    return k.to(DTYPES[c["dtype"]]), v.to(DTYPES[c["dtype"]])


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
    k, v = (x.transpose(0, 1) for x in _plain_values(s, s["pages"][kseq, kpos // P].long(), kpos % P))      # [kv heads][keys][D]
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


def _columns(s):
    """The settings as columns over the rows."""
    rows = s["case"]["rows"]
    return tuple(torch.as_tensor(s[w], device="cuda").double().expand(rows)[:, None] for w in ("temperature", "top_k", "top_p", "min_p"))


def _plain_sample(s):
    # in 64 bits: a running sum over a whole vocabulary lies next to the border of some token
    temperature, top_k, top_p, min_p = _columns(s)
    x, order = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True)
    greedy = temperature <= 0
    w = torch.exp((x - x[:, :1]) / torch.where(greedy, torch.ones_like(temperature), temperature))
    place = torch.arange(x.shape[1], device="cuda")
    within = place < torch.where(top_k > 0, top_k, torch.full_like(top_k, math.inf))
    w = w * within
    before = torch.cumsum(w, -1) - w
    keep = within & ((before < top_p * w.sum(-1, keepdim=True)) | (top_p >= 1)) & (w >= min_p) & ~greedy | (place == 0)
    w = torch.zeros_like(w).scatter_(1, order, w * keep)
    run = torch.cumsum(w, -1)
    token = (run > s["uniform"].double()[:, None] * run[:, -1:]).int().argmax(-1)
    chance = w.gather(1, token[:, None])[:, 0] / run[:, -1]
    return token, torch.log(chance).float()


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"append": _plain_append, "load": _plain_load, "mha": _plain_mha, "sample": _plain_sample}[c["op"]](s)
    if c["op"] == "sample":
        from eet_b200 import EET
        return EET.sample_rows(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                               min_p=s["min_p"])
    from eet_b200 import paged
    table = (s["pages"], s["starts"], s["lens"])
    if c["op"] == "mha":
        return paged.paged_mha(s["q"], s["k_cache"], s["v_cache"], *table, max_tokens=s["max_tokens"], max_len=s["max_len"],
                               window=c["window"], first_key=s["first_key"], alibi_slopes=s["alibi_slopes"],
                               k_scale=s["k_scale"], v_scale=s["v_scale"])
    q = None
    if c["op"] == "append":
        q = paged.paged_store(s["k"], s["v"], s["k_cache"], s["v_cache"], *table, q=s["q"], freqs=s["freqs"],
                              interleaved=c["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    k, v = paged.paged_load(s["k_cache"], s["v_cache"], *table, s["tokens"], dtype=DTYPES[c["dtype"]], k_scale=s["k_scale"],
                            v_scale=s["v_scale"])
    return (k, v) if q is None else (q, k, v, s["k_scale"], s["v_scale"])


# ---------------------------------------------------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------------------------------------------------
def _turn64(x, position, s):
    """Pair i of a row as a complex number, turned by exp(i position freqs[i])."""
    x, half = x.double(), s["freqs"].numel()
    phase = torch.polar(torch.ones(len(x), half, dtype=torch.float64, device="cuda"), torch.outer(position.double(), s["freqs"]))[:, None]
    y = x.clone()
    places = torch.arange(2 * half, device="cuda")
    one, two = (places[0::2], places[1::2]) if s["case"]["interleaved"] else (places[:half], places[half:2 * half])
    z = torch.complex(x[..., one], x[..., two]) * phase
    y[..., one], y[..., two] = z.real, z.imag
    return y


def _nearest64(y, codes):
    """The values that a row of head dim stands for once it is quantised, and its scale, which is kept in 32 bits."""
    dtype, most = CODES[codes]
    scale = (y.abs().max(-1, keepdim=True).values / most).float().double()
    scale[scale == 0] = 1.0
    # the codes' magnitudes in their order, and the nearest, or of two that are as near the even one
    table = torch.arange(128, dtype=torch.uint8, device=y.device)
    table = table.double() if codes == "int8" else table[:127].view(dtype).double()
    borders = (table[1:] + table[:-1]) / 2
    z = (y / scale).abs()
    at = torch.bucketize(z, borders)
    at += (z == borders[at.clamp(max=len(borders) - 1)]) & (at % 2 == 1)
    return table[at.clamp(max=len(table) - 1)] * y.sign() * scale, scale[..., 0]


def _exact_append(s, new, lens):
    c, at, parts = s["case"], 0, ([], [], [])
    scales = [s["k_scale"].double(), s["v_scale"].double()]
    for b, n in enumerate(new):
        place = torch.arange(lens[b] - n, lens[b], device="cuda")
        page = s["pages"][b].long()[place // c["page"]]
        rows = slice(at, at + n)
        parts[0].append(_turn64(s["q"][rows], place, s))
        for i, y in enumerate((_turn64(s["k"][rows], place, s), s["v"][rows].double())):
            y, scales[i][page, :, place % c["page"]] = _nearest64(y, c["codes"])
            parts[1 + i].append(y)
        at += n
    return tuple(torch.cat(p) for p in parts) + tuple(scales)


def _exact_sample(s):
    c = s["case"]
    settings = [x[:, 0].tolist() for x in _columns(s)]
    tokens, chances = [], []
    for row, x in enumerate(s["logits"].double()):
        t, k, p, m = (column[row] for column in settings)
        best = x.argsort(descending=True, stable=True)
        if t <= 0:
            tokens.append(int(best[0]))
            chances.append(0.0)
            continue
        best = best[:int(k)] if 0 < k < c["vocab"] else best
        prob = torch.softmax(x[best] / t, 0)
        ends = torch.cat((prob.new_zeros(1), prob.cumsum(0)))
        kept = min(int((ends[:-1] < p).sum()) if p < 1 else len(best), int((prob >= m * prob[0]).sum()))
        kept = best[:max(1, kept)].sort().values
        prob = torch.softmax(x[kept] / t, 0)
        at = min(int((prob.cumsum(0) <= s["uniform"][row].double()).sum()), len(kept) - 1)
        tokens.append(int(kept[at]))
        chances.append(float(torch.log(prob[at])))
    return torch.tensor(tokens, device="cuda"), torch.tensor(chances, dtype=torch.float64, device="cuda")


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    new, lens, first = _lengths(case)
    P, at = case["page"], 0
    if case["op"] == "append":
        return _exact_append(s, new, lens)
    if case["op"] == "load":
        parts = [], []
        for b, n in enumerate(new):
            place = torch.arange(lens[b] - n, lens[b], device="cuda")
            page = s["pages"][b].long()[place // P]
            for i, w in enumerate("kv"):
                parts[i].append(s[w + "_cache"][page, :, place % P].double() * s[w + "_scale"][page, :, place % P].double()[..., None])
        return tuple(torch.cat(p) for p in parts)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    G, D = case["heads"] // case["kv_heads"], case["head_dim"]
    for b, n in enumerate(new):
        place = torch.arange(lens[b], device="cuda")
        page = s["pages"][b].long()[place // P]
        for h in range(case["kv_heads"]):
            k, v = (s[w + "_cache"][page, h, place % P].double() * s[w + "_scale"][page, h, place % P].double()[:, None] for w in "kv")
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
