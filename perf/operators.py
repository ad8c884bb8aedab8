"""Workloads of the class-score and per-leaf product operators on one GPU.

Four kinds of work, each one call of a program that boosts, scores or fits models of many classes:

* ``log_probs``       - ``ops.class_log_probs``: raw class scores [rows, classes] become the log probability of a given class,
  the log of the normaliser, the entropy and the top alternatives of every row.
* ``log_probs_grad``  - ``ops.class_log_probs_grad``: the gradient in the scores of a loss made of those quantities.
* ``leaf_products``   - ``ops.leaf_products``: rows grouped by leaf, each leaf with its own linear map to several outputs.
* ``leaf_grad``       - the gradients of that product in its rows (``ops.leaf_products`` with the transposed maps) and in its
  maps (``ops.leaf_gram``, which also gives the normal equations of linear leaves).

Scores lie in memory by row (what ``Booster.predict`` returns) or by class (the training scores that a custom objective sees).
"""
from __future__ import annotations

import math
from typing import Any, Dict, List

import numpy as np
import torch

own = False

_LOGP = {"kind": "log_probs", "rows": 1, "classes": 2, "dtype": "float32", "layout": "row", "top": 0, "unlabelled": 0.0, "masked": 0.0, "spread": 2.5}
_LEAF = {"kind": "leaf_products", "rows": 1, "features": 28, "outputs": 10, "leaves": 31, "dtype": "float32"}


def listed() -> List[Dict[str, Any]]:
    return [
        # The scores of one request of an online service: a handful of rows, ten classes, the three best answers. Latency only.
        dict(_LOGP, name="log_probs_request", rows=16, classes=10, top=3),
        # The training scores of a ten-class table as a custom objective or metric sees them: class-major, full precision.
        dict(_LOGP, name="log_probs_train_scores", rows=1_000_000, classes=10, layout="class", top=2, spread=1.5),
        # One row over a large set of classes (a catalogue, a vocabulary): the row has to be split to use the machine.
        dict(_LOGP, name="log_probs_one_row", rows=1, classes=131_072, dtype="bfloat16", top=20),
        # A batch over an odd number of classes, a fifth of them ruled out by -inf (some rows lose all), some rows without a label.
        dict(_LOGP, name="log_probs_masked", rows=4_099, classes=50_021, dtype="float16", top=5, unlabelled=0.05, masked=0.2),
        # The largest batch over the large set of classes.
        dict(_LOGP, name="log_probs_batch", rows=4_096, classes=131_072, dtype="bfloat16", top=20),
        # Gradients of a custom objective (likelihood and entropy) on the training scores of the ten-class table.
        dict(_LOGP, name="grad_train_scores", kind="log_probs_grad", rows=1_000_000, classes=10, layout="class", unlabelled=0.05, spread=1.5),
        # The same loss, with the top alternatives in it, over many classes in a half type.
        dict(_LOGP, name="grad_batch", kind="log_probs_grad", rows=8_191, classes=32_001, dtype="bfloat16", top=5, unlabelled=0.05),
        # A small batch through the linear leaves of one tree: 136 features, as in the ranking shape. Latency only.
        dict(_LEAF, name="leaf_request", rows=64, features=136, outputs=10, leaves=31),
        # The headline benchmark's 28 features and 255 leaves, ten outputs, a million rows: a matter of bandwidth.
        dict(_LEAF, name="leaf_narrow", rows=1_000_000, features=28, outputs=10, leaves=255),
        # Two thousand features to a thousand classes: a matter of the tensor cores.
        dict(_LEAF, name="leaf_wide", rows=65_536, features=2_000, outputs=1_000, leaves=63, dtype="bfloat16"),
        # Gradients of the narrow form: the shape in which linear leaves are fitted.
        dict(_LEAF, name="leaf_grad_narrow", kind="leaf_grad", rows=1_000_000, features=28, outputs=10, leaves=255),
        # Gradients of a wide form in the other half type, an odd number of rows and outputs.
        dict(_LEAF, name="leaf_grad_wide", kind="leaf_grad", rows=50_001, features=1_000, outputs=513, leaves=15, dtype="float16"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> Dict[str, Any]:
    """One more case of the ranges above, sizes spread over their logarithms."""
    while True:
        kind = rng.choice(["log_probs", "log_probs", "log_probs_grad", "leaf_products", "leaf_grad"])
        dtype = rng.choice(["float32", "bfloat16", "float16"])
        if kind.startswith("log"):
            case = dict(_LOGP, kind=kind, dtype=dtype, rows=_log_int(rng, 1, 2_000_000), classes=_log_int(rng, 2, 200_000), layout=rng.choice(["row", "row", "class"]),
                        unlabelled=rng.choice([0.0, 0.1]), masked=rng.choice([0.0, 0.0, 0.3]), spread=rng.choice([1.5, 2.5, 6.0]))
            case["top"] = min(case["classes"], rng.choice([0, 1, 2, 3, 5, 10, 20, 32]))
            if case["layout"] == "class":
                case["classes"] = min(case["classes"], 2_000)   # boosting keeps one tree per class and round
                case["top"] = min(case["classes"], case["top"])
            if case["rows"] * case["classes"] <= 300_000_000:
                return case
        else:
            case = dict(_LEAF, kind=kind, dtype=dtype, rows=_log_int(rng, 1, 2_000_000), features=_log_int(rng, 4, 2_000), outputs=_log_int(rng, 1, 1_000), leaves=_log_int(rng, 2, 255))
            wide = case["rows"] * (case["features"] + case["outputs"])
            product = case["rows"] * case["features"] * case["outputs"]
            if wide <= 150_000_000 and case["leaves"] * case["features"] * case["outputs"] <= 150_000_000 and product <= (1.3e11 if dtype != "float32" else 1e10) / (2 if kind == "leaf_grad" else 1):
                return case


# ---------------------------------------------------------------------------------------------------- inputs ----
def _seed(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _leaf_sizes(case: Dict[str, Any], seed: int) -> np.ndarray:
    """Rows of every leaf: a few large leaves, many middling ones, some that no row of this data reaches."""
    r = np.random.RandomState(seed % (1 << 31))
    share = r.gamma(2.0, size=case["leaves"])
    if case["leaves"] >= 8:
        share[r.choice(case["leaves"], size=case["leaves"] // 16 + 1, replace=False)] = 0.0
    return r.multinomial(case["rows"], share / share.sum())


def prepare(case: Dict[str, Any], seed: int) -> Dict[str, Any]:
    g, dtype, n = _seed(seed), getattr(torch, case["dtype"]), case["rows"]
    state: Dict[str, Any] = {"case": case}
    if case["kind"].startswith("log"):
        k = case["classes"]
        by_class = case["layout"] == "class"
        scores = torch.randn((k, n) if by_class else (n, k), generator=g, device="cuda", dtype=dtype).mul_(case["spread"])
        if case["masked"]:
            out = torch.rand(scores.shape, generator=g, device="cuda", dtype=torch.float16) < case["masked"]
            out |= (torch.rand(n, generator=g, device="cuda") < 0.002).unsqueeze(0 if by_class else 1)   # rows that lose every class
            scores.masked_fill_(out, -math.inf)
            del out
        labels = torch.randint(0, k, (n,), generator=g, device="cuda", dtype=torch.int32)
        if case["unlabelled"]:
            labels[torch.rand(n, generator=g, device="cuda") < case["unlabelled"]] = -1
        state.update(scores=scores.t() if by_class else scores, labels=labels)
        if case["kind"] == "log_probs_grad":
            # a program has the results of the forward call in hand, and the gradients that its loss sends back
            p = _log_probs(state["scores"], labels, case["top"])
            state.update(log_norm=p["log_norm"], entropy=p["entropy"], top_class=p.get("top_class"))
            state.update(g_log_prob=torch.randn(n, generator=g, device="cuda"), g_entropy=torch.randn(n, generator=g, device="cuda") * 0.1,
                         g_log_norm=torch.randn(n, generator=g, device="cuda") * 0.1,
                         g_top=torch.randn((n, case["top"]), generator=g, device="cuda") * 0.1 if case["top"] else None)
    else:
        sizes = _leaf_sizes(case, seed)
        begin = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        f, k, leaves = case["features"], case["outputs"], case["leaves"]
        state.update(x=torch.randn((n, f), generator=g, device="cuda", dtype=dtype),
                     weight=torch.randn((leaves, k, f), generator=g, device="cuda", dtype=dtype).mul_(f ** -0.5),
                     begin=torch.from_numpy(begin).cuda(), most=int(sizes.max()))
        if case["kind"] == "leaf_grad":
            state["grad"] = torch.randn((n, k), generator=g, device="cuda", dtype=dtype)
    return state


# ---------------------------------------------------------------------------------------------------- plain ----
def _top_classes(s: torch.Tensor, top: int):
    """Classes by falling score, equal scores by rising class: one whole number per class holds both. (torch: [rows, top])"""
    k = s.shape[1]
    bits = (s + 0.0).contiguous().view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    keys = (bits.long() << 32) | torch.arange(k - 1, -1, -1, device=s.device)
    found = torch.topk(keys, top, dim=1, sorted=True).values
    return (k - 1) - (found & 0xFFFFFFFF)


def _log_probs(scores: torch.Tensor, labels: torch.Tensor, top: int) -> Dict[str, torch.Tensor]:
    s = scores.float()
    most = s.max(dim=1).values
    none = most == -math.inf
    most = torch.where(none, torch.zeros_like(most), most)
    x = s - most[:, None]
    e = torch.exp(x)
    total = e.sum(dim=1)
    log_norm = most + torch.log(total)
    mean = torch.where(e > 0, e * x, torch.zeros_like(e)).sum(dim=1) / total
    entropy = torch.where(none, torch.zeros_like(mean), torch.log(total) - mean)
    given = s.gather(1, labels.long().clamp(min=0)[:, None])[:, 0]
    log_prob = torch.where(given == -math.inf, given, given - log_norm)
    out = {"log_prob": torch.where(labels < 0, torch.zeros_like(log_prob), log_prob), "log_norm": log_norm, "entropy": entropy}
    if top:
        c = _top_classes(s, top)
        v = s.gather(1, c)
        out["top_log_prob"] = torch.where(v == -math.inf, v, v - log_norm[:, None])
        out["top_class"] = torch.where(v == -math.inf, torch.full_like(c, -1), c).int()
    return out


def _log_probs_grad(st: Dict[str, Any]) -> torch.Tensor:
    s, labels, top = st["scores"].float(), st["labels"].long(), st["top_class"]
    labelled = labels >= 0
    none = st["log_norm"] == -math.inf
    lp = s - torch.where(none, torch.zeros_like(st["log_norm"]), st["log_norm"])[:, None]
    p = torch.exp(lp)
    g_lp = torch.where(labelled, st["g_log_prob"], torch.zeros_like(st["g_log_prob"]))
    a = st["g_log_norm"] - g_lp - st["g_entropy"] * st["entropy"]
    if top is not None:
        g_top = torch.where(top >= 0, st["g_top"], torch.zeros_like(st["g_top"]))
        a = a - g_top.sum(dim=1)
    grad = torch.where(p > 0, p * (a[:, None] - st["g_entropy"][:, None] * lp), torch.zeros_like(p))
    grad.scatter_add_(1, labels.clamp(min=0)[:, None], g_lp[:, None])
    if top is not None:
        grad.scatter_add_(1, top.long().clamp(min=0), g_top)
    grad = torch.where(none[:, None], torch.zeros_like(grad), grad)
    return grad.to(st["scores"].dtype)


def _places(st: Dict[str, Any], n: int):
    """Rows of every leaf side by side, [leaves, most], whether each is there, and where each row then is."""
    begin, most = st["begin"].long(), max(1, st["most"])
    at = begin[:-1, None] + torch.arange(most, device=begin.device)
    there = at < begin[1:, None]
    rows = torch.arange(n, device=begin.device)
    leaf = torch.searchsorted(begin, rows, right=True) - 1
    return at.clamp(max=n - 1), there, leaf * most + rows - begin[leaf]


def _leaf_products(x: torch.Tensor, weight: torch.Tensor, places) -> torch.Tensor:
    at, _, back = places
    y = torch.bmm(x.float()[at], weight.float().transpose(1, 2))
    return y.reshape(-1, weight.shape[1])[back].to(x.dtype)


def _leaf_gram(a: torch.Tensor, b: torch.Tensor, places) -> torch.Tensor:
    at, there, _ = places
    return torch.bmm((a.float()[at] * there[:, :, None]).transpose(1, 2), b.float()[at]).to(a.dtype)


# ---------------------------------------------------------------------------------------------------- run ----
def run(st: Dict[str, Any]) -> Any:
    kind = st["case"]["kind"]
    if own:
        from falcata_b200 import ops

        if kind == "log_probs":
            r = ops.class_log_probs(st["scores"], st["labels"], top_k=st["case"]["top"])
            return {name: value for name, value in r._asdict().items() if value is not None}
        if kind == "log_probs_grad":
            return ops.class_log_probs_grad(st["scores"], st["log_norm"], st["entropy"], labels=st["labels"], top_class=st["top_class"], grad_log_prob=st["g_log_prob"],
                                            grad_log_norm=st["g_log_norm"], grad_entropy=st["g_entropy"], grad_top_log_prob=st["g_top"])
        if kind == "leaf_products":
            return ops.leaf_products(st["x"], st["weight"], st["begin"])
        return [ops.leaf_products(st["grad"], st["weight"].transpose(1, 2), st["begin"]), ops.leaf_gram(st["grad"], st["x"], st["begin"])]
    if kind == "log_probs":
        return _log_probs(st["scores"], st["labels"], st["case"]["top"])
    if kind == "log_probs_grad":
        return _log_probs_grad(st)
    places = _places(st, st["case"]["rows"])
    if kind == "leaf_products":
        return _leaf_products(st["x"], st["weight"], places)
    return [_leaf_products(st["grad"], st["weight"].transpose(1, 2), places), _leaf_gram(st["grad"], st["x"], places)]


def work(case: Dict[str, Any]) -> Dict[str, float]:
    n, size = case["rows"], 4 if case["dtype"] == "float32" else 2
    if case["kind"].startswith("log"):
        k, top = case["classes"], case["top"]
        per_row = 4 + 3 * 4 + 8 * top                       # label, three results, alternatives
        if case["kind"] == "log_probs":
            return {"bytes": n * (k * size + per_row), "flops": 5.0 * n * k}
        return {"bytes": n * (2 * k * size + per_row + 8), "flops": 5.0 * n * k}
    f, k, leaves = case["features"], case["outputs"], case["leaves"]
    once = size * (n * f + n * k + leaves * k * f) + 4 * (leaves + 1)
    if case["kind"] == "leaf_products":
        return {"bytes": once, "flops": 2.0 * n * f * k}
    return {"bytes": once + size * (n * f + leaves * k * f), "flops": 4.0 * n * f * k}


# ---------------------------------------------------------------------------------------------------- exact ----
def exact(case: Dict[str, Any], seed: int) -> Any:
    st = prepare(case, seed)
    if case["kind"].startswith("log"):
        return _exact_scores(case, st)
    return _exact_leaves(case, st)


def _exact_scores(case: Dict[str, Any], st: Dict[str, Any]) -> Any:
    n, k, top = case["rows"], case["classes"], case["top"]
    step = max(1, 50_000_000 // k)
    parts = []
    for lo in range(0, n, step):
        s = st["scores"][lo:lo + step].double()
        y = st["labels"][lo:lo + step].long()
        lse = torch.logsumexp(s, dim=1)
        none = torch.isneginf(lse)
        logp = torch.where(torch.isneginf(s), s, s - lse[:, None])
        p = torch.where(torch.isneginf(logp), 0.0, torch.exp(logp))
        plogp = torch.where(p > 0, p * logp, 0.0)
        h = -plogp.sum(1)
        rows = torch.arange(s.shape[0], device=s.device)
        if case["kind"] == "log_probs":
            got = [torch.where(y < 0, 0.0, logp[rows, y.clamp(min=0)]), lse, h]
            if top:
                # a stable sort puts equal scores in the order of their classes
                _, c = torch.sort(s, dim=1, descending=True, stable=True)
                c = c[:, :top]
                v = logp.gather(1, c)
                got += [v, torch.where(torch.isneginf(v), -1, c).int()]
            parts.append(got)
            continue
        g_lp = torch.where(y < 0, 0.0, st["g_log_prob"][lo:lo + step].double())
        g_h, g_z = st["g_entropy"][lo:lo + step].double(), st["g_log_norm"][lo:lo + step].double()
        # d logp_c / d s_j = [c == j] - p_j;  d lse / d s_j = p_j;  d H / d s_j = -p_j (log p_j + H)
        d = g_z[:, None] * p - g_h[:, None] * (plogp + p * h[:, None]) - g_lp[:, None] * p
        d[rows, y.clamp(min=0)] += g_lp
        if top:
            c = st["top_class"][lo:lo + step].long()
            g_t = torch.where(c < 0, 0.0, st["g_top"][lo:lo + step].double())
            d -= g_t.sum(1)[:, None] * p
            d.scatter_add_(1, c.clamp(min=0), g_t)
        parts.append([torch.where(none[:, None], 0.0, d)])
    whole = [torch.cat(x) for x in zip(*parts)]
    if case["kind"] == "log_probs_grad":
        return whole[0]
    return dict(zip(["log_prob", "log_norm", "entropy", "top_log_prob", "top_class"], whole))


def _exact_leaves(case: Dict[str, Any], st: Dict[str, Any]) -> Any:
    begin = st["begin"].cpu().tolist()
    x, w = st["x"].double(), st["weight"].double()
    spans = list(zip(begin[:-1], begin[1:]))
    if case["kind"] == "leaf_products":
        return torch.cat([x[lo:hi] @ w[leaf].t() for leaf, (lo, hi) in enumerate(spans)])
    d = st["grad"].double()
    return [torch.cat([d[lo:hi] @ w[leaf] for leaf, (lo, hi) in enumerate(spans)]), torch.stack([d[lo:hi].t() @ x[lo:hi] for lo, hi in spans])]
