"""The op set of the IR: for every op its kind, operand count, result shape
rule and NumPy meaning.

The names, attributes, kinds and result shapes are Kiln's (the reference's
kiln/ir/ops.py:48-188); the fusion pass, buffer assignment and the HIP
lowering dispatch on the kind. The NumPy meaning serves the constant folder
at compile time and ``interpret`` (a whole-graph evaluator for pass tests);
nothing on the GPU path calls it.

Kinds: ``elementwise`` (shapes broadcast NumPy-style), ``reduction``
(``dims``, always keepdim), ``matmul`` ([B,] M x K @ [B,] K x N), ``view``
(transpose / reshape / slice / expand: no data movement once buffers are
assigned), ``paged`` (the operators over a paged key/value cache, which the
reference does not have) and ``const``.
"""

from __future__ import annotations

import math

import numpy as np

from kiln.ir.core import Graph, TensorType


class OpSpec:
    """kind, arity (None = any), shape(in_shapes, attrs) -> out shape or None,
    compute(arrays, attrs) -> array."""

    __slots__ = ("name", "kind", "arity", "shape", "compute")

    def __init__(self, name, kind, arity, shape, compute):
        self.name, self.kind, self.arity, self.shape, self.compute = name, kind, arity, shape, compute

    # kept for callers that read the fields by their older names
    infer = property(lambda self: self.shape)
    ref = property(lambda self: self.compute)


OPS: dict = {}


def _add(name, kind, arity, shape, compute):
    OPS[name] = OpSpec(name, kind, arity, shape, compute)


def broadcast_shapes(*shapes) -> tuple:
    return tuple(np.broadcast_shapes(*shapes))


# -- elementwise --------------------------------------------------------------------

_SQRT_2_OVER_PI = math.sqrt(2.0 / math.pi)
_erf_f64 = np.vectorize(math.erf, otypes=[np.float64])


def gelu_reference(x, approximate="none"):
    """GELU evaluated in float64: x * Phi(x), or with approximate="tanh"
    0.5 x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3)))."""
    x = np.asarray(x, dtype=np.float64)
    if approximate == "tanh":
        inner = _SQRT_2_OVER_PI * (x + 0.044715 * x * x * x)
        return 0.5 * x * (1.0 + np.tanh(inner))
    return 0.5 * x * (1.0 + _erf_f64(x * (1.0 / math.sqrt(2.0))))


def _unary(x, attrs, op):
    if op == "neg":
        return -x
    if op == "exp":
        return np.exp(x)
    if op == "tanh":
        return np.tanh(x)
    if op == "sigmoid":
        return 1.0 / (1.0 + np.exp(-x))
    if op == "relu":
        return np.maximum(x, 0)
    if op == "gelu":
        return gelu_reference(x, attrs.get("approximate", "none"))
    if op == "rsqrt":
        return 1.0 / np.sqrt(x)
    if op == "sqrt":
        return np.sqrt(x)
    if op == "erf":
        return _erf_f64(x)
    if op == "copy":
        return np.array(x, copy=True)
    raise KeyError(op)


_BINARY_UFUNC = {"add": np.add, "sub": np.subtract, "mul": np.multiply, "div": np.divide,
                 "maximum": np.maximum, "minimum": np.minimum}
UNARY_OPS = ("neg", "exp", "tanh", "sigmoid", "relu", "gelu", "rsqrt", "sqrt", "erf", "copy")
BINARY_OPS = tuple(_BINARY_UFUNC)


def _broadcast_rule(shapes, attrs):
    return broadcast_shapes(*shapes)


for _op in UNARY_OPS:
    _add(_op, "elementwise", 1, _broadcast_rule, lambda xs, attrs, _op=_op: _unary(xs[0], attrs, _op))
for _op, _ufunc in _BINARY_UFUNC.items():
    _add(_op, "elementwise", 2, _broadcast_rule, lambda xs, attrs, _u=_ufunc: _u(xs[0], xs[1]))


# -- reductions (keepdim) ---------------------------------------------------------------

def _reduced_shape(shapes, attrs):
    (shape,) = shapes
    rank = len(shape)
    gone = {d % rank for d in attrs["dims"]} if rank else set()
    return tuple(1 if d in gone else extent for d, extent in enumerate(shape))


_add("reduce_sum", "reduction", 1, _reduced_shape,
     lambda xs, attrs: xs[0].sum(axis=tuple(attrs["dims"]), keepdims=True))
_add("reduce_max", "reduction", 1, _reduced_shape,
     lambda xs, attrs: xs[0].max(axis=tuple(attrs["dims"]), keepdims=True))

# the elementwise op that combines two partial results, and its identity
REDUCTION_COMBINER = {"reduce_sum": "add", "reduce_max": "maximum"}
REDUCTION_INIT = {"reduce_sum": 0.0, "reduce_max": float("-inf")}


# -- matmul ---------------------------------------------------------------------------------

def _matmul_shape(shapes, attrs):
    a, b = shapes
    batch_ok = len(a) == len(b) and a[:-2] == b[:-2]
    if not (batch_ok and len(a) in (2, 3) and a[-1] == b[-2]):
        raise ValueError(f"matmul: incompatible shapes {a} x {b}")
    return tuple(a[:-1]) + (b[-1],)


_add("matmul", "matmul", 2, _matmul_shape, lambda xs, attrs: xs[0] @ xs[1])


# -- views ------------------------------------------------------------------------------------

def _transpose_shape(shapes, attrs):
    src = shapes[0]
    return tuple(src[axis] for axis in attrs["perm"])


def _reshape_shape(shapes, attrs):
    target = tuple(attrs["shape"])
    if math.prod(target) != math.prod(shapes[0]):
        raise ValueError(f"reshape: {shapes[0]} -> {target} changes element count")
    return target


def _slice_shape(shapes, attrs):
    dims = list(shapes[0])
    d = attrs["dim"] % len(dims)
    lo, hi, step = attrs["start"], min(attrs["end"], dims[d]), attrs.get("step", 1)
    dims[d] = len(range(lo, hi, step)) if hi > lo else 0
    return tuple(dims)


def _slice_compute(xs, attrs):
    x = xs[0]
    index = tuple(slice(attrs["start"], attrs["end"], attrs.get("step", 1)) if d == attrs["dim"] % x.ndim
                  else slice(None) for d in range(x.ndim))
    return x[index]


_add("transpose", "view", 1, _transpose_shape, lambda xs, attrs: np.transpose(xs[0], attrs["perm"]))
_add("reshape", "view", 1, _reshape_shape, lambda xs, attrs: np.reshape(xs[0], tuple(attrs["shape"])))
_add("slice", "view", 1, _slice_shape, _slice_compute)
_add("expand", "view", 1, lambda shapes, attrs: broadcast_shapes(shapes[0], tuple(attrs["shape"])),
     lambda xs, attrs: np.broadcast_to(xs[0], tuple(attrs["shape"])))

# -- the paged cache (kiln/hip/paged.py says what the operators compute) -----------------------

# paged_attention: q, k, v, k_pages, v_pages, table, lengths[, parents][, selected]
#   {scale, cache (element type of the pages), parents, selected (whether given)}
# select_pages: q, k_means, table, lengths {page_size, pages}


def _paged_attention_shape(shapes, attrs):
    q, k, v, k_pages, v_pages, table, lengths = shapes[:7]
    given = 7 + bool(attrs["parents"]) + bool(attrs["selected"])
    s, n, heads, dim = q
    kv = k_pages[1]
    ok = (len(shapes) == given and v_pages == k_pages and k_pages[3] == dim and k == v == (s, n, kv, dim)
          and kv and heads % kv == 0 and table[0] == s and lengths == (s,))
    if ok and attrs["parents"]:
        ok = shapes[7] == (s, n)
    if ok and attrs["selected"]:
        ok = shapes[given - 1][:3] == (s, n, kv)
    if not ok:
        raise ValueError(f"paged_attention: shapes {shapes} do not fit each other")
    return q


def _select_pages_shape(shapes, attrs):
    q, means, table, lengths = shapes
    if not (means[2] == q[3] and means[1] and q[2] % means[1] == 0 and table[0] == q[0] and lengths == q[:1]):
        raise ValueError(f"select_pages: shapes {shapes} do not fit each other")
    return q[0], q[1], means[1], attrs["pages"]


def _rounded(x, dtype):
    if dtype == "f16":
        return x.astype(np.float16).astype(np.float64)
    if dtype == "bf16":   # nearest, ties to even
        u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
        u = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16 << 16).astype(np.uint32)
        return np.where(np.isnan(x), np.nan, u.view(np.float32)).astype(np.float64)
    return x.astype(np.float64)


def _paths(parents, n):
    """The tokens each drafted token sees, or None where it is unused."""
    out = []
    for i in range(n):
        up = i - 1 if parents is None else int(parents[i])
        before = [] if up == -1 else out[up] if 0 <= up < i else None
        out.append(None if before is None else before + [i])
    return out


def _paged_attention(xs, attrs):
    q, k, v, k_pages, v_pages, table, lengths = xs[:7]
    parents = xs[7] if attrs["parents"] else None
    selected = xs[-1] if attrs["selected"] else None
    batch, n, heads, dim = q.shape
    pages, kv, ps, _ = k_pages.shape
    new_k, new_v = _rounded(k, attrs["cache"]), _rounded(v, attrs["cache"])
    out = np.zeros(q.shape)
    for s in range(batch):
        length = max(0, min(int(lengths[s]), table.shape[1] * ps))
        for i, path in enumerate(_paths(None if parents is None else parents[s], n)):
            if path is None:
                continue
            for h in range(heads):
                c = h // (heads // kv)
                columns = range(table.shape[1])
                if selected is not None:
                    row = [-1, *map(int, selected[s, i, c])]
                    columns = [b for a, b in zip(row, row[1:]) if b > a and 0 <= b < table.shape[1]]
                spots = [(int(table[s, b]), min(ps, length - b * ps)) for b in columns if b * ps < length]
                spots = [(p, m) for p, m in spots if 0 <= p < pages]
                keys = np.concatenate([k_pages[p, c, :m] for p, m in spots] + [new_k[s, path, c]]).astype(np.float64)
                values = np.concatenate([v_pages[p, c, :m] for p, m in spots] + [new_v[s, path, c]]).astype(np.float64)
                score = keys @ q[s, i, h].astype(np.float64) * attrs["scale"]
                e = np.exp(score - score.max())
                out[s, i, h] = e @ values / e.sum()
    return out


def _select_pages(xs, attrs):
    q, means, table, lengths = xs
    batch, n, heads, _ = q.shape
    total, kv, _ = means.shape
    ps, top = attrs["page_size"], attrs["pages"]
    out = np.full((batch, n, kv, top), -1, np.int32)
    for s in range(batch):
        held = -(-max(0, min(int(lengths[s]), table.shape[1] * ps)) // ps)
        for i in range(n):
            for c in range(kv):
                group = q[s, i, c * (heads // kv):(c + 1) * (heads // kv)].astype(np.float64).sum(0)
                score = [float(group @ means[p, c].astype(np.float64)) if 0 <= (p := int(table[s, b])) < total else 0.0
                         for b in range(held)]
                order = sorted(range(held), key=lambda b: (b != held - 1, math.isnan(score[b]),
                                                           0.0 if math.isnan(score[b]) else -score[b], b))
                best = sorted(order[:top])
                out[s, i, c, :len(best)] = best
    return out


_add("paged_attention", "paged", None, _paged_attention_shape, _paged_attention)
_add("select_pages", "paged", 4, _select_pages_shape, _select_pages)

# operands of the paged operators that are the cache itself: its pages, tables and
# lists, read where they lie (never copied or converted), and given anew each call
PAGED_OPERANDS = {"paged_attention": 3, "select_pages": 1}   # the first such operand
RESULT_TYPE = {"select_pages": "i32"}


# const: its type is always given explicitly, its data comes from the graph
_add("const", "const", 0, lambda shapes, attrs: None, lambda xs, attrs: None)


# -- queries ------------------------------------------------------------------------------------

def kind(op: str) -> str:
    return OPS[op].kind


def infer_type(op: str, input_types, attrs) -> TensorType:
    spec = OPS.get(op)
    if spec is None:
        raise ValueError(f"unknown op '{op}'")
    if spec.arity is not None and len(input_types) != spec.arity:
        raise ValueError(f"{op} expects {spec.arity} operands, got {len(input_types)}")
    if spec.kind not in ("view", "paged") and any(t.dtype != "f32" for t in input_types):
        raise ValueError(f"{op}: operands must be f32")
    if spec.kind == "paged":
        _check_paged_types(op, input_types, attrs)
    shape = spec.shape([t.shape for t in input_types], attrs)
    if shape is None:
        raise ValueError(f"{op}: result type must be given explicitly")
    dtype = input_types[0].dtype if spec.kind == "view" else RESULT_TYPE.get(op, "f32")
    return TensorType(tuple(map(int, shape)), dtype)


def _check_paged_types(op, types, attrs):
    if op == "select_pages":
        wanted = [("f32", 4), ("f32", 3), ("i32", 2), ("i32", 1)]
    else:
        cache = attrs["cache"]
        wanted = [("f32", 4)] * 3 + [(cache, 4)] * 2 + [("i32", 2), ("i32", 1)]
        wanted += [("i32", 2)] * bool(attrs["parents"]) + [("i32", 4)] * bool(attrs["selected"])
    if [(t.dtype, t.rank) for t in types] != wanted:
        raise ValueError(f"{op}: operands {', '.join(map(str, types))} do not fit the operator")


def evaluate(op: str, inputs, attrs) -> np.ndarray:
    """One op on NumPy arrays; always returns a C-contiguous float32 array
    (0-d for a scalar result; int32 for a list of pages)."""
    result = OPS[op].compute([np.asarray(x) for x in inputs], attrs)
    whole = RESULT_TYPE.get(op) == "i32" or (kind(op) == "view" and np.asarray(inputs[0]).dtype == np.int32)
    return np.array(result, dtype=np.int32 if whole else np.float32, order="C")


def interpret(graph: Graph, *inputs) -> list:
    """Evaluate the whole graph with the NumPy meaning of each op. ``inputs``
    feed the non-``param`` arguments in order; ``param`` arguments read their
    data from ``graph.constants``."""
    runtime = [i for i, attrs in enumerate(graph.arg_attrs) if "param" not in attrs]
    if len(inputs) != len(runtime):
        raise ValueError(f"expected {len(runtime)} inputs, got {len(inputs)}")
    values = {}
    for arg, attrs in zip(graph.args, graph.arg_attrs):
        if "param" in attrs:
            values[arg] = graph.constants[attrs["param"]]
    for i, x in zip(runtime, inputs):   # (16-bit pages come as the float32 values they hold)
        values[graph.args[i]] = np.asarray(x, np.int32 if graph.args[i].type.dtype == "i32" else np.float32)
    for node in graph.nodes:
        if node.op == "const":
            values[node.out] = graph.const_data(node.out)
        else:
            values[node.out] = evaluate(node.op, [values[v] for v in node.inputs], node.attrs)
    return [values[v] for v in graph.results]
