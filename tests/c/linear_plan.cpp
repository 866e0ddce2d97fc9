// The cuts that csrc/linear_plan.h chooses, for tests: one call a line on stdin, one JSON object a line on stdout.  Needs no GPU.
//   product elem I J P a_dma b_dma
//   forward dtype m n k ldx ldw
//   backward dtype act x_act packed m n k ldg ldx ldw gradients     (gradients: a sum of 1 gx, 2 gw, 4 gb)
// Operands lie at 16-byte addresses.
#include <iostream>
#include <sstream>
#include <string>

#include "linear_plan.h"

static void print(const char *name, const Cut &c)
{
    std::cout << "\"" << name << "\": {\"tile\": " << (64 << c.tile) << ", \"tiles\": " << c.tiles_i * c.tiles_j << ", \"whole\": " << c.whole
              << ", \"splits\": " << c.splits << ", \"a_dma\": " << c.a_dma << ", \"b_dma\": " << c.b_dma << "}, ";
}

int main()
{
    char *const at = (char *)(1 << 20);
    for (std::string line; std::getline(std::cin, line);) {
        std::istringstream in(line);
        std::string what;
        in >> what;
        std::cout << "{";
        if (what == "product") {
            int elem, a, b;
            int64_t I, J, P;
            in >> elem >> I >> J >> P >> a >> b;
            print("product", plan_product(elem, I, J, P, a, b));
            std::cout << "\"total\": 0";
        } else if (what == "forward") {
            pifu_linear_args g{};
            in >> g.dtype >> g.m >> g.n >> g.k >> g.ldx >> g.ldw;
            g.x = g.w = g.y = at;
            g.ldy = g.n;
            const Forward f = plan_forward(g);
            print("product", f.cut);
            std::cout << "\"copies\": " << (f.ldx != 0) + (f.ldw != 0) << ", \"total\": " << f.total;
        } else {
            pifu_linear_grad_args g{};
            int packed, gradients;
            in >> g.dtype >> g.act >> g.x_act >> packed >> g.m >> g.n >> g.k >> g.ldg >> g.ldx >> g.ldw >> gradients;
            g.grad = g.w = at;
            if (packed) g.x8.codes = g.x8.scales = g.z8.codes = g.z8.scales = (uint8_t *)at;
            else g.x = g.z = at;
            if (gradients & 1) g.gx = at;
            if (gradients & 2) g.gw = at;
            if (gradients & 4) g.gb = at;
            const Plan p = plan_backward(g);
            if (g.gx) print("gx", p.gx);
            if (g.gw) print("gw", p.gw);
            std::cout << "\"halves\": " << p.halves_dz + 2 * p.halves_h << ", \"scaled\": " << p.scaled << ", \"narrow\": " << p.narrow << ", \"copies\": " << (p.ldw != 0) << ", \"total\": " << p.total;
        }
        std::cout << "}" << std::endl;
    }
    return 0;
}
