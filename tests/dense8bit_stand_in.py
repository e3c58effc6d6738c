"""The 8-bit dense layer's kernels on the CPU, in place of the binding that `dense_ops` calls: for tests of the layer."""
import torch

BLOCK = 128


class Binding:
    def quantize_blocks(self, x, rows):
        r, k = x.shape
        v = torch.nn.functional.pad(x.float(), (0, -k % BLOCK, 0, -r % rows)).view(-(-r // rows), rows, -(-k // BLOCK), BLOCK)
        part, power = torch.frexp(v.abs().amax((1, 3)).clamp(min=2.0 ** -126))
        scales = torch.ldexp(torch.ones_like(part), power - 9 + (part > 0.875).int())
        codes = (v / scales[:, None, :, None]).to(torch.float8_e4m3fn)
        return codes.reshape(-(-r // rows) * rows, -1)[:r, :k].contiguous(), scales

    def dense_8bit(self, x, kernel, scales, bias, residual, activation, check):
        from tf_approximate_b200 import InvalidArgumentError
        if scales.dtype != torch.float32 or kernel.dtype != torch.float8_e4m3fn or x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise InvalidArgumentError("types")
        if residual is not None and residual.dtype != x.dtype:
            raise InvalidArgumentError("residual")
        units, inputs = kernel.shape
        with torch.no_grad():
            q, s = self.quantize_blocks(x.reshape(-1, inputs), 1)
            a = q.float() * s.repeat_interleave(BLOCK, 1)[:, :inputs]
            w = kernel.float() * scales.repeat_interleave(BLOCK, 0)[:units].repeat_interleave(BLOCK, 1)[:, :inputs]
            z = (a @ w.t()).view(*x.shape[:-1], units)
            for more in (bias, residual):
                z = z if more is None else z + more.float()
            return (lambda v: v, torch.relu, torch.nn.functional.gelu, torch.nn.functional.silu)[activation](z).to(x.dtype)


def place(monkeypatch):
    from tf_approximate_b200 import dense_ops
    monkeypatch.setattr(dense_ops._lib, "binding", Binding)
