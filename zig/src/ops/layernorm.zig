//! Layer norm over the last dimension with a gain and a bias vector, as an op module (not compiled
//! in this repository).
//!
//!   forward   u_i = mean_j x[i, j],   r_i = 1 / sqrt(mean_j (x[i, j] - u_i)^2 + eps)
//!             h[i, j] = (x[i, j] - u_i) * r_i,   z[i, j] = h[i, j] * g[j] + b[j]
//!   reverse   e[i, j] = z.grad[i, j] * g[j]
//!             x.grad[i, j] += r_i * (e[i, j] - mean_j e[i, j] - h[i, j] * mean_j(e[i, j] * h[i, j]))
//!             g.grad[j]    += sum_i z.grad[i, j] * h[i, j],   b.grad[j] += sum_i z.grad[i, j]
//!
//! x is taken as [m, n] with n its last size; g and b have n elements. The sums over the rows are
//! added in a fixed order, so g.grad and b.grad do not depend on scheduling. The reverse's workspace
//! comes from the stream's scratch (src/core/utils.zig:20-36), sized by mpLayernormReverseScratchBytes.
const std = @import("std");
const core = @import("core");
const OpDatum = core.OpDatum;
const Tensor = core.Tensor;
const Graph = core.Graph;
const dev = core.utils.dev;

fn last_size(t: Tensor) usize {
    const s = t.sizes();
    std.debug.assert(s.len >= 1);
    return s[s.len - 1];
}

// an index counts within its class (src/core/graph.zig:34-41)
fn same(a: Tensor, b: Tensor) bool {
    return a.ptr == b.ptr and a.idx == b.idx and a.class == b.class;
}

pub fn forward(x: Tensor, gain: Tensor, bias: Tensor, eps: f64) Tensor {
    return forward_impl(x.ptr, x, gain, bias, eps);
}

pub fn forward_impl(graph: *Graph, x: Tensor, gain: Tensor, bias: Tensor, eps: f64) Tensor {
    const n = last_size(x);
    std.debug.assert(gain.len() == n);
    std.debug.assert(gain.dtype() == x.dtype());
    std.debug.assert(bias.len() == n);
    std.debug.assert(bias.dtype() == x.dtype());
    // one launch writes the three gradients
    std.debug.assert(!same(x, gain));
    std.debug.assert(!same(x, bias));
    std.debug.assert(!same(gain, bias));
    const m = if (n == 0) 0 else x.len() / n;

    const out = graph.tensor(.{ .class = .hid, .dtype = x.dtype(), .sizes = x.sizes() });
    const key = core.dkey(out);

    core.invoke(core.kernels.layernorm_ij_j, key, .{
        x.data_ptr(), gain.data_ptr(), bias.data_ptr(), out.data_ptr(), eps, m, n, out.context(),
    });

    if (graph.mode == .train) {
        core.attach_op(@This(), out, &.{
            OpDatum{ .tensor = x },
            OpDatum{ .tensor = gain },
            OpDatum{ .tensor = bias },
            OpDatum{ .scalar = eps },
            OpDatum{ .tensor = out },
        });
    }
    return out;
}

pub fn reverse(args: []const OpDatum) void {
    const x = args[0].tensor;
    const gain = args[1].tensor;
    const bias = args[2].tensor;
    const eps = args[3].scalar;
    const out = args[4].tensor;
    core.enable_gradient(x);
    core.enable_gradient(gain);
    core.enable_gradient(bias);

    const n = last_size(x);
    const m = if (n == 0) 0 else x.len() / n;
    const key = core.dkey(out);

    // never zero bytes for a non-empty problem: the partial rows go through it
    const bytes = dev.mpLayernormReverseScratchBytes(key, m, n);
    const scratch = out.stream().get_scratch(.r32, (bytes + 3) / 4);
    core.invoke(core.kernels.layernorm_ij_j_reverse, key, .{
        x.data_ptr(), gain.data_ptr(), out.grad_ptr(), x.grad_ptr(), gain.grad_ptr(), bias.grad_ptr(),
        scratch, eps, @as(f64, 1.0), m, n, out.context(),
    });
}

pub fn derive(_: []const OpDatum, _: Tensor) ?OpDatum {
    return null;
}
